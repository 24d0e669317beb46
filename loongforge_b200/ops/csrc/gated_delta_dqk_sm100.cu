// dQ and dK of the gated delta rule for head dims dk = dv = 128, on tcgen05 (gated_delta_sm100.cu has the formulas).
//
// One (chunk, value head) is five products with 128 rows and 128 columns in TMEM. Tokens are rows, 0-63 for dq and
// 64-127 for dk (or for what leads there):
//
//   D3 = [dO; dV] [U; u]^T + [0; v] [U; u]^T        -> W = strict_lower(dO U^T) D and N = -strict_lower(dV U^T) D, in two parts each
//   D1 = [dO; dV] (S0 + s0)^T + [0; v] S0^T         -> dq += e^G (.), dk -= e^G (.)
//   D2 = [  ; U] (dS1 + ds1)^T + [  ; u] dS1^T      -> dk += e^{G_C - G} (.)
//   D4 = [W; N] K + [0; W^T] Q + [0; N^T] K         -> dq += , dk +=
//
// with capitals for the bf16 high parts and v, u, s0, ds1 for what they leave of dV, U and the states; products of two such
// remainders are left out (2^-18 of the term). The diagonal of W comes from the backward chain and is added to the rows in
// fp32 at the end. Rows are scaled when the accumulators are read, so that every operand is a
// bf16 tile as it lies in memory. An operand tile whose first 64 rows are not wanted starts 64 rows early: what lies there
// ends in rows of D2 that nobody reads; where they have to be zeros, v, W and N lie columns first, so that their first 64
// rows can come from a tile of zeros elsewhere.
//
// 208 KB a (chunk, value head) come in, 128 of them the two states in two parts each, and 48 a (chunk, key head): about
// 290 us at 16384 tokens, 16 key and 32 value heads, where the kernel takes 540 (144 at 4096). With the high parts of S0, dS1
// and dV alone it took 358 (97), and dq and dk were off by 2.4e-3 where decays are near one, instead of the 1.66e-3 of their
// rounding. One block per SM goes through its share of (chunk, key head) pairs; seven warps bring tiles (fragments of
// registers, turned by stmatrix on the way), one thread issues the products, eight warps make W and N, and add up rows over
// the value heads of a key head. The tiles fill shared memory: a state's low part takes the place of its high part when the
// products have read that, and a unit's loads begin when its predecessor's products are done. What bounds it are these two
// rounds of loads, which alternate with the products: 19K cycles a unit.
#include <atomic>
#include "gated_delta.cuh"
#include "sm100_ptx.cuh"

namespace lf {
namespace {

using namespace delta;

// Warps 0-7 compute, 8-14 load, 15 issues: sixteen warps leave 128 registers a thread, seventeen 96.
constexpr int D = 128, LOAD_WARPS = 7, LOADERS = 32 * LOAD_WARPS, THREADS = 512;
// 16 x 16 fragments of one 128 x 128 operand, of one 128 x 64, and a warp's shares
constexpr int TILES = 64, MINE = (TILES + LOAD_WARPS - 1) / LOAD_WARPS, VTILES = 32, VMINE = (VTILES + LOAD_WARPS - 1) / LOAD_WARPS;
constexpr uint32_t BIG = 128 * 128, BOX = 64 * 128;                    // bytes of a 128 x 64 and a 64 x 64 box

struct Smem {
  unsigned char xo[2 * BIG], xu[2 * BIG], s0[2 * BIG], ds[2 * BIG];  // [dO; dV], [U_hi; U_lo]; [v][dk] of both states
  unsigned char q[2 * BOX], k[2 * BOX], zero[BOX], w[4 * BOX], v[2 * BOX];  // w: W_hi, N_hi, W_lo, N_lo; v: [v][token]
  float vec[2][DELTA_VEC];
  float dots[2][128];
  uint64_t xos_full, ds_full, s0_free, ds_free, s0_low, ds_low, qk_full, tiles_free, qk_free, d3_done, w_ready, d4_done, acc_free;
  uint32_t tmem;
};
enum { T_D1 = 0, T_D2 = 128, T_D3 = 256, T_D4 = 384 };

// Byte offset of the 16-byte piece c of row r in a swizzled box.
__device__ __forceinline__ uint32_t piece_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// A [128 rows][K] K-major in boxes of `abox` bytes, B [128 rows][K] K-major / [K][128 columns] in boxes of `bbox`.
template <int KS>
__device__ __forceinline__ void mma_kk(uint32_t d, uint32_t a, uint32_t abox, uint32_t b, uint32_t bbox, bool more) {
  constexpr uint32_t idesc = make_idesc(1, 1, false, false, 128, 128);
#pragma unroll
  for (int s = 0; s < KS; ++s)
    tc_mma_f16_ss(d, make_smem_desc_sw128(a + (s >> 2) * abox + (s & 3) * 32, 16, 1024), make_smem_desc_sw128(b + (s >> 2) * bbox + (s & 3) * 32, 16, 1024), idesc, more || s > 0);
}
template <int KS>
__device__ __forceinline__ void mma_km(uint32_t d, uint32_t a, uint32_t abox, uint32_t b, uint32_t bbox, bool more) {
  constexpr uint32_t idesc = make_idesc(1, 1, false, true, 128, 128);
#pragma unroll
  for (int s = 0; s < KS; ++s)
    tc_mma_f16_ss(d, make_smem_desc_sw128(a + (s >> 2) * abox + (s & 3) * 32, 16, 1024), make_smem_desc_sw128(b + s * 2048, bbox, 1024), idesc, more || s > 0);
}
// A^T with A [16 KS rows of K][64 columns] behind 64 columns of zeros, of which 64 rows serve for all; added to D.
template <int KS>
__device__ __forceinline__ void mma_tm(uint32_t d, uint32_t zero, uint32_t a, uint32_t b, uint32_t bbox) {
  constexpr uint32_t idesc = make_idesc(1, 1, true, true, 128, 128);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const uint32_t z = zero + (s & 3) * 2048;
    tc_mma_f16_ss(d, make_smem_desc_sw128(z, a + s * 2048 - z, 1024), make_smem_desc_sw128(b + s * 2048, bbox, 1024), idesc, 1u);
  }
}
template <int KS>
__device__ __forceinline__ void mma_tk(uint32_t d, uint32_t zero, uint32_t a, uint32_t b, uint32_t bbox) {
  constexpr uint32_t idesc = make_idesc(1, 1, true, false, 128, 128);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const uint32_t z = zero + (s & 3) * 2048;
    tc_mma_f16_ss(d, make_smem_desc_sw128(z, a + s * 2048 - z, 1024), make_smem_desc_sw128(b + (s >> 2) * bbox + (s & 3) * 32, 16, 1024), idesc, 1u);
  }
}

__device__ __forceinline__ void stsm(uint32_t addr, const uint4& r) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
}
__device__ __forceinline__ void stsm_t(uint32_t addr, const uint4& r) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
}

// The two parts of eight fp32 values of U.
__device__ __forceinline__ void split_u(const uint4& x, const uint4& y, uint4& hi, uint4& lo) {
  split2(__uint_as_float(x.x), __uint_as_float(x.y), hi.x, lo.x);
  split2(__uint_as_float(x.z), __uint_as_float(x.w), hi.y, lo.y);
  split2(__uint_as_float(y.x), __uint_as_float(y.y), hi.z, lo.z);
  split2(__uint_as_float(y.z), __uint_as_float(y.w), hi.w, lo.w);
}

// The block's (chunk, key head) pairs, every gridDim.x-th, without a division each.
struct Item {
  int c, hk, dc, dh;
  __device__ __forceinline__ explicit Item(const DeltaArgs& a) {
    c = static_cast<int>(blockIdx.x) / a.Hk;
    hk = static_cast<int>(blockIdx.x) - c * a.Hk;
    dc = static_cast<int>(gridDim.x) / a.Hk;
    dh = static_cast<int>(gridDim.x) - dc * a.Hk;
  }
  __device__ __forceinline__ void next(const DeltaArgs& a) {
    c += dc;
    hk += dh;
    if (hk >= a.Hk) {
      hk -= a.Hk;
      ++c;
    }
  }
};

// Sixteen neighbouring values of a factor row.
__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 f = reinterpret_cast<const float4*>(p)[i];
    x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
  }
}

__global__ void __launch_bounds__(THREADS, 1)
tc_dqk_kernel(const DeltaArgs a) {
  extern __shared__ unsigned char raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw + (1024 - (smem_addr(raw) & 1023)) % 1024);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rep = a.Hv / a.Hk;
  if (threadIdx.x == 0) {
    bar_init(&sm.xos_full, LOAD_WARPS);
    bar_init(&sm.ds_full, LOAD_WARPS);
    bar_init(&sm.s0_free, 1);
    bar_init(&sm.ds_free, 1);
    bar_init(&sm.s0_low, LOAD_WARPS);
    bar_init(&sm.ds_low, LOAD_WARPS);
    bar_init(&sm.qk_full, LOAD_WARPS);
    bar_init(&sm.tiles_free, 1);
    bar_init(&sm.qk_free, 8);
    bar_init(&sm.d3_done, 1);
    bar_init(&sm.w_ready, 8);
    bar_init(&sm.d4_done, 1);
    bar_init(&sm.acc_free, 8);
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < static_cast<int>(sizeof(sm.zero) / 16); i += THREADS) reinterpret_cast<uint4*>(sm.zero)[i] = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  if (warp == 15) tmem_alloc(&sm.tmem, 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tm = sm.tmem;
  // u counts the (chunk, value head) pairs of the block, i the (chunk, key head) pairs; every role goes the same way
  int u = 0, i = 0;

  if (warp < 8) {
    const int quarter = warp & 3, half = warp >> 2, r = 32 * quarter + lane, tok = r & 63;
    const bool key = r >= 64;
    const uint32_t lanes = tm + (static_cast<uint32_t>(32 * quarter) << 16);
    const uint32_t wt = smem_addr(sm.w);
    for (Item it(a); it.c < a.NC; it.next(a)) {
      const int c = it.c, hk = it.hk;
      const Span sp = chunk_span(a, c);
      if (sp.len == 0) continue;
      float acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0.f;
      float norm = 1.f, wd = 0.f;  // wd: the diagonal of W in the thread's row
      for (int hr = 0; hr < rep; ++hr, ++u) {
        const float* vec = sm.vec[u & 1];
        // W_ij = qs_i rk_j D_ij (dO U^T)_ij, N_ij = -rk_i rk_j D_ij (dV U^T)_ij, i > j
        bar_wait(&sm.d3_done, u & 1, a.status);
        tc_fence_after_sync();
        const float gh = vec[V_GHI * 64 + tok], gl = vec[V_GLO * 64 + tok];
        const float f = key ? -vec[V_RK * 64 + tok] : vec[V_QS * 64 + tok];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          // element by element the chain of latencies is long: sixteen at a time, made everywhere and selected at the end
          const int j0 = 32 * half + 16 * b;
          float e[16], x[16];
          load16(vec + V_GHI * 64 + j0, e);
          load16(vec + V_GLO * 64 + j0, x);
#pragma unroll
          for (int j = 0; j < 16; ++j) e[j] = __expf((gh - e[j]) + (gl - x[j]));
          load16(vec + V_RK * 64 + j0, x);
#pragma unroll
          for (int j = 0; j < 16; ++j) e[j] *= f * x[j];
          uint32_t y[16], ph[8], pl[8];
          tmem_ld_32x32b_x16(lanes + T_D3 + j0, y);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = __uint_as_float(y[j]);
          tmem_ld_32x32b_x16(lanes + T_D3 + 64 + j0, y);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            e[j] *= x[j] + __uint_as_float(y[j]);
            e[j] = j0 + j < tok ? e[j] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) split2(e[2 * j], e[2 * j + 1], ph[j], pl[j]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t at = piece_at(r, 4 * half + 2 * b + j);
            *reinterpret_cast<uint4*>(sm.w + at) = make_uint4(ph[4 * j], ph[4 * j + 1], ph[4 * j + 2], ph[4 * j + 3]);
            *reinterpret_cast<uint4*>(sm.w + 2 * BOX + at) = make_uint4(pl[4 * j], pl[4 * j + 1], pl[4 * j + 2], pl[4 * j + 3]);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        bar_arrive(&sm.w_ready);
        wd += w_diagonal(a, static_cast<long long>(c) * a.Hv + hk * rep + hr, tok, vec);
        // the rows, scaled; D1 and D2 while D4 is under way
        const float f1 = key ? -vec[V_YK * 64 + tok] : vec[V_OQ * 64 + tok], f2 = vec[V_SU * 64 + tok];
        norm = vec[(key ? V_RK : V_RQ) * 64 + tok];
        bar_wait(&sm.tiles_free, u & 1, a.status);
        tc_fence_after_sync();
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t x[16];
          tmem_ld_32x32b_x16(lanes + T_D1 + 64 * half + 16 * b, x);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[16 * b + j] += f1 * __uint_as_float(x[j]);
          if (key) {  // a whole warp or none of it
            tmem_ld_32x32b_x16(lanes + T_D2 + 64 * half + 16 * b, x);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[16 * b + j] += f2 * __uint_as_float(x[j]);
          }
        }
        tc_fence_before_sync();
        bar_arrive(&sm.acc_free);  // now the next head's vec may replace this one's, and the next products these
        bar_wait(&sm.d4_done, u & 1, a.status);
        tc_fence_after_sync();
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t x[16];
          tmem_ld_32x32b_x16(lanes + T_D4 + 64 * half + 16 * b, x);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[16 * b + j] += __uint_as_float(x[j]);
        }
      }
      // The rows are r dq^ and r dk^ with r = 1 / norm, so that dq = r dq^ - q r^2 (q . r dq^), the same for k.
      const unsigned char *tile = key ? sm.k : sm.q, *other = key ? sm.q : sm.k;
      bar_wait(&sm.qk_full, i & 1, a.status);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint4 y = *reinterpret_cast<const uint4*>(other + half * BOX + piece_at(tok, j));
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[8 * j + 2 * e] += wd * lo_half(w[e]);
          acc[8 * j + 2 * e + 1] += wd * hi_half(w[e]);
        }
      }
      uint4 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const uint4*>(tile + half * BOX + piece_at(tok, j));
      float f = 0.f;
      if (a.l2norm) {
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) d += acc[8 * j + 2 * e] * lo_half(w[e]) + acc[8 * j + 2 * e + 1] * hi_half(w[e]);
        }
        sm.dots[half][r] = d;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        f = (sm.dots[0][r] + sm.dots[1][r]) * norm * norm;
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      // through w's place, which only these warps write, to whole rows
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2(acc[8 * j + 2 * e] - f * lo_half(w[e]), acc[8 * j + 2 * e + 1] - f * hi_half(w[e]));
        *reinterpret_cast<uint4*>(sm.w + half * BIG + piece_at(r, j)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      bar_arrive(&sm.qk_free);
      asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 16 * warp + 2 * j + (lane >> 4), p = lane & 15, t = row & 63;
        if (t < sp.len)
          *reinterpret_cast<uint4*>(static_cast<bf16*>(row < 64 ? a.dq : a.dkey) + ((sp.start + t) * a.Hk + hk) * D + p * 8) =
              *reinterpret_cast<const uint4*>(sm.w + (p >> 3) * BIG + piece_at(row, p & 7));
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      ++i;
    }
  } else if (warp < 15) {
    const int lw = warp - 8, tid = threadIdx.x - 256;
    const int m = lane >> 3, l8 = lane & 7;
    const uint32_t xu = smem_addr(sm.xu), s0 = smem_addr(sm.s0), ds = smem_addr(sm.ds), vl = smem_addr(sm.v);
    for (Item it(a); it.c < a.NC; it.next(a)) {
      const int c = it.c, hk = it.hk;
      const Span sp = chunk_span(a, c);
      if (sp.len == 0) continue;
      for (int hr = 0; hr < rep; ++hr, ++u) {
        const int h = hk * rep + hr;
        const long long rec = static_cast<long long>(c) * a.Hv + h;
        // U, in fp32: 8 tiles of columns x 4 of tokens x 2; v the same, one each; the states: 8 tiles of columns x 2 parts x 8 of dk
        uint4 fu[MINE], fs[MINE];
        const uint4* us = reinterpret_cast<const uint4*>(a.u) + rec * 8 * 256 + lane;
        const uint4* vs = reinterpret_cast<const uint4*>(a.dv_lo) + rec * 8 * 128 + lane;
        const uint4* ss = reinterpret_cast<const uint4*>(a.states) + rec * 8 * 512 + lane;
        const uint4* dd = reinterpret_cast<const uint4*>(a.dstates) + rec * 8 * 512 + lane;
        auto take_state = [&](uint4 (&f)[MINE], const uint4* src, int part) {
#pragma unroll
          for (int j = 0; j < MINE; ++j) {
            const int t = lw + LOAD_WARPS * j;
            if (t < TILES) f[j] = src[(t >> 3) * 512 + part * 256 + (t & 7) * 32];
          }
        };
        auto put_state = [&](uint32_t dst, const uint4 (&f)[MINE]) {
#pragma unroll
          for (int j = 0; j < MINE; ++j) {
            const int t = lw + LOAD_WARPS * j, v = 16 * (t >> 3) + (m & 1) * 8 + l8, k = 16 * (t & 7) + (m >> 1) * 8;
            if (t < TILES) stsm(dst + (k >> 6) * BIG + piece_at(v, (k >> 3) & 7), f[j]);
          }
        };
#pragma unroll
        for (int j = 0; j < VMINE; ++j) {
          const int t = lw + LOAD_WARPS * j;
          if (t < VTILES) {
            fu[2 * j] = us[64 * t];
            fu[2 * j + 1] = us[64 * t + 32];
          }
        }
        take_state(fs, ss, 0);
        // the last head's products have read the tiles; D1 of it waited until the vec of two heads ago was read
        if (u > 0) bar_wait(&sm.tiles_free, (u - 1) & 1, a.status);
        const long long row = (sp.start * a.Hv + h) * D, stride = static_cast<long long>(a.Hv) * D;
        {  // [dO; dV]: a thread takes one 16-byte column of every 14th row
          const int p = tid & 15;
          unsigned char* dst = sm.xo + (p >> 3) * BIG;
#pragma unroll 1
          for (int part = 0; part < 2; ++part) {
            const bf16* src = static_cast<const bf16*>(part ? a.dv_ : a.dout) + row + p * 8;
#pragma unroll 1
            for (int t = tid >> 4; t < 64; t += LOADERS / 16) cp16(dst + piece_at(64 * part + t, p & 7), src + (t < sp.len ? t * stride : 0), t < sp.len);
          }
        }
        if (tid < DELTA_VEC / 4) cp16(&sm.vec[u & 1][tid * 4], a.vec + rec * DELTA_VEC + tid * 4, true);
        cp_commit();
#pragma unroll
        for (int j = 0; j < VMINE; ++j) {
          const int f = lw + LOAD_WARPS * j, t = 16 * (f & 3) + (m >> 1) * 8 + l8, v = 16 * (f >> 2) + (m & 1) * 8;
          const uint32_t at = xu + (v >> 6) * BIG + piece_at(t, (v >> 3) & 7);
          uint4 hi, lo;
          split_u(fu[2 * j], fu[2 * j + 1], hi, lo);
          if (f < VTILES) {
            stsm_t(at, hi);
            stsm_t(at + BOX, lo);  // 64 rows further on
          }
        }
#pragma unroll
        for (int j = 0; j < VMINE; ++j) {
          const int t = lw + LOAD_WARPS * j;
          if (t < VTILES) fu[j] = vs[32 * t];
        }
        put_state(s0, fs);
#pragma unroll
        for (int j = 0; j < VMINE; ++j) {
          const int f = lw + LOAD_WARPS * j, v = 16 * (f >> 2) + (m & 1) * 8 + l8;
          if (f < VTILES) stsm(vl + piece_at(v, 2 * (f & 3) + (m >> 1)), fu[j]);
        }
        cp_wait<0>();
        fence_proxy_async_smem();  // before the loads below: it waits for loads in flight too
        bar_arrive(&sm.xos_full);
        take_state(fu, dd, 0);
        take_state(fs, ss, 1);
        put_state(ds, fu);
        fence_proxy_async_smem();
        bar_arrive(&sm.ds_full);
        take_state(fu, dd, 1);
        if (hr == 0) {
          if (i > 0) bar_wait(&sm.qk_free, (i - 1) & 1, a.status);
          const bf16* qp = static_cast<const bf16*>(a.q) + sp.start * a.q_ts + hk * a.q_hs;
          const bf16* kp = static_cast<const bf16*>(a.k) + sp.start * a.k_ts + hk * a.k_hs;
          const int p = tid & 15;
#pragma unroll 1
          for (int r = tid >> 4; r < 64; r += LOADERS / 16) {
            const bool ok = r < sp.len;
            const uint32_t at = (p >> 3) * BOX + piece_at(r, p & 7);
            cp16(sm.q + at, qp + (ok ? r * a.q_ts : 0) + p * 8, ok);
            cp16(sm.k + at, kp + (ok ? r * a.k_ts : 0) + p * 8, ok);
          }
          cp_commit();
          cp_wait<0>();
          fence_proxy_async_smem();
          bar_arrive(&sm.qk_full);
        }
        // the states' low parts, where the high ones have been read
        bar_wait(&sm.s0_free, u & 1, a.status);
        put_state(s0, fs);
        fence_proxy_async_smem();
        bar_arrive(&sm.s0_low);
        bar_wait(&sm.ds_free, u & 1, a.status);
        put_state(ds, fu);
        fence_proxy_async_smem();
        bar_arrive(&sm.ds_low);
      }
      ++i;
    }
  } else {
    if (lane == 0) {
      const uint32_t xo = smem_addr(sm.xo), xu = smem_addr(sm.xu), s0 = smem_addr(sm.s0), ds = smem_addr(sm.ds);
      const uint32_t q = smem_addr(sm.q), k = smem_addr(sm.k), zero = smem_addr(sm.zero), w = smem_addr(sm.w), v = smem_addr(sm.v);
      for (Item it(a); it.c < a.NC; it.next(a)) {
        if (chunk_span(a, it.c).len == 0) continue;
        for (int hr = 0; hr < rep; ++hr, ++u) {
          const uint32_t parity = u & 1;
          bar_wait(&sm.xos_full, parity, a.status);
          tc_fence_after_sync();
          mma_kk<8>(tm + T_D3, xo, BIG, xu, BIG, false);  // W of the last head was made before its D4 was issued
          mma_tk<8>(tm + T_D3, zero, v, xu, BIG);
          tc_commit(&sm.d3_done);
          if (u > 0) bar_wait(&sm.acc_free, (u - 1) & 1, a.status);
          tc_fence_after_sync();
          mma_km<8>(tm + T_D1, xo, BIG, s0, BIG, false);
          mma_tm<8>(tm + T_D1, zero, v, s0, BIG);
          tc_commit(&sm.s0_free);
          bar_wait(&sm.ds_full, parity, a.status);
          tc_fence_after_sync();
          mma_km<8>(tm + T_D2, xu - BOX, BIG, ds, BIG, false);
          mma_km<8>(tm + T_D2, xu, BIG, ds, BIG, true);
          tc_commit(&sm.ds_free);
          bar_wait(&sm.s0_low, parity, a.status);
          tc_fence_after_sync();
          mma_km<8>(tm + T_D1, xo, BIG, s0, BIG, true);
          bar_wait(&sm.ds_low, parity, a.status);
          tc_fence_after_sync();
          mma_km<8>(tm + T_D2, xu - BOX, BIG, ds, BIG, true);
          tc_commit(&sm.tiles_free);
          if (hr == 0) bar_wait(&sm.qk_full, i & 1, a.status);
          bar_wait(&sm.w_ready, parity, a.status);
          tc_fence_after_sync();
          mma_km<4>(tm + T_D4, w, 0, k, BOX, false);
          mma_km<4>(tm + T_D4, w + 2 * BOX, 0, k, BOX, true);
          mma_tm<4>(tm + T_D4, zero, w, q, BOX);
          mma_tm<4>(tm + T_D4, zero, w + 2 * BOX, q, BOX);
          mma_tm<4>(tm + T_D4, zero, w + BOX, k, BOX);
          mma_tm<4>(tm + T_D4, zero, w + 3 * BOX, k, BOX);
          tc_commit(&sm.d4_done);
        }
        ++i;
      }
    }
    __syncwarp();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 15) {
    tc_fence_after_sync();
    tmem_dealloc(tm, 512);
  }
}

}  // namespace

int delta_tc_dqk(const DeltaArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  const size_t bytes = sizeof(Smem) + 1024;
  if (!allow_smem(tc_dqk_kernel, bytes, allowed)) return -3;
  const long long items = a.NC * a.Hk, sms = sm_count();
  tc_dqk_kernel<<<static_cast<unsigned>(items < sms ? items : sms), THREADS, bytes, s>>>(a);
  return 0;
}

}  // namespace lf
