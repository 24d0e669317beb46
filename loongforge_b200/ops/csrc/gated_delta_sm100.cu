// Gated delta rule over chunks of 64 tokens, forward and backward.
//
// With q, k normalised (q scaled), G the running sum of the log decays inside a chunk, D_ij = exp(G_i - G_j), S0 the
// state the chunk starts from ([dk, dv]) and rows = tokens:
//
//   M = strict_lower(beta_i (k_i.k_j) D_ij),   A = (I + M)^-1,   P = lower((q_i.k_j) D_ij)
//   U = A diag(beta) (V - diag(e^G) K S0),     O = diag(e^G) Q S0 + P U,     S1 = e^{G_C} S0 + K^T diag(e^{G_C - G}) U
//
// and, from dO and dS1,
//
//   X = A^T (P^T dO + diag(e^{G_C - G}) K dS1),   dV = diag(beta) X,   dbeta = (X . U) / beta
//   dS0 = e^{G_C} dS1 + Q^T diag(e^G) dO - K^T diag(e^G) dV
//   dQ = diag(e^G) dO S0^T + W K,   W = lower(dO U^T) D   (its diagonal, do_i.u_i, apart and in fp32)
//   dK = -diag(e^G) dV S0^T + diag(e^{G_C - G}) U dS1^T + W^T Q + (N + N^T) K,   N = -strict_lower(dV U^T) D
//
// The gradient of a log decay g_t gathers what every token or state in front of t gives to every token or state from t
// on. With o~_i the part of o_i, and m_i = v_i - u_i / beta_i the part of the memory read at i, that earlier tokens
// wrote, and x~_j the part of X_j that later tokens ask for,
//
//   dg_t = sum_{i >= t} (o~_i.do_i - m_i.dv_i) - sum_{j >= t} u_j.x~_j + sum_j e^{G_C - G_j} (K dS1)_j.u_j + e^{G_C} <dS1, S0>
//
// with sums over the chunk. Every term carries a decay, so heads that decay strongly throughout keep the relative accuracy
// of their (small) gradient; that is why A and P are kept as strict lower parts, their diagonals apart: o~, m and x~ are
// sums of their own, never differences of larger numbers. That does not hold for a single reset among mild decays: a pair
// j < i of tokens that both lie behind t enters dg_t once through o~_i and m_i and once, negated, through x~_j, and neither
// carries g_t. What is left of such a dg_t is the rounding of its neighbours' terms (3e-7 where they are of order one, as
// with fp32 products).
//
// Kernels:
//   prepare   one block per (chunk, key head): Q K^T and K K^T once, then A, P and the per-token factors of each of its
//             value heads.
//   forward   walks along the sequence. The delta rule acts on every column of dv by itself, so 16 columns of a head make
//             a unit that never waits for another one. All products are transposed: S^T [16, dk] lies in accumulators of
//             mma.sync, and an accumulator tile is, register by register, the A operand of the next product. Four warps
//             share a unit (by dk for the state, by tokens for the rest) and hand their operands to each other.
//   backward  the same in reverse with dS^T.
//   dqk       dQ and dK, parallel over chunks: in gated_delta_dqk_sm100.cu for dk = dv = 128, here where either is 64.
//   gates     dg and dbeta.
//
// Precision. Sums and the state are fp32. An fp32 operand of a product is cut into bf16 parts: r, U and its scaled copy, dU
// and P into three (24 bits), since they make up the results as they are; the state, A, dS1 and what is added to it into two:
// a decay lies between what they leave out, 2^-18, and the results, which makes it small unless it is near one; and dQ and
// dK take two parts of everything but the diagonal of W, which is far below their rounding. Products of parts below 2^-24
// are left out. The third parts of P lie in the blocks of its tiles that no product reads, those of r, U and dU in shared
// memory of their own; they cost 22 us forward of what stands below at 4096 tokens. With the gates of a new layer states, dg
// and dbeta come out within 1e-7, 5e-7 and 1.4e-7 (2-norm; 2e-6 to 6e-6 with two parts everywhere), as with fp32 products;
// with decays of 1e-3 a token, within 2e-6, 4e-6 and 4e-6. Exponentials are the fast ones: 2^-22 of a decay near one, and
// 2^-20 of e^-10.
//
// The chain is bound by latency: three dependent products of at most 64 x 128 x 16 per chunk, with a hand-over between
// them, 6.5K cycles a chunk forward and 8K backward. mma.sync runs at a quarter of tcgen05's rate, but operands and results
// stay in registers, and 32 heads make 1024 warps of such work. One sequence of 4096 tokens with 32 heads of 128 x 128 (five
// sequences of 16384): prepare 39 us (137), forward 212 (740), backward 261 (886), dqk 144 (540), gates 8 (16); 190 (656)
// and 238 (826) before the third parts and the low ones that dqk reads. Measured against that: a whole unit in one warp 471
// (959) forward and 620 (1278) backward; eight warps along the chain and eight beside it 208 (713) and 257 (874), bound by
// shared memory; a head as one 128-column product on tcgen05 11.7K cycles a chunk, 5K of them the work on elements between
// the products, on an eighth as many blocks.
#include "gated_delta.cuh"

namespace lf {
namespace {

using namespace delta;
constexpr int APITCH = 72;  // bf16 per row of a 64-wide tile: odd multiple of 16 bytes, no bank conflicts in ldmatrix

// ------------------------------------------------------------------------------------------------------- primitives

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], const bf16* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], const bf16* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_addr(p)) : "memory");
}
__device__ __forceinline__ void stsm_t(bf16* p, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(smem_addr(p)), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// Addresses of the lane for the four 8x8 tiles of one x4 load, p = row-major base, `ld` its pitch. With m = lane / 8:
// tile m covers rows r0 + 8 * (m & 1), columns c0 + 8 * (m >> 1)
__device__ __forceinline__ const bf16* at_rc(const bf16* p, int ld, int r0, int c0) {
  const int l = threadIdx.x & 31, m = l >> 3;
  return p + (r0 + (m & 1) * 8 + (l & 7)) * ld + c0 + (m >> 1) * 8;
}
// tile m covers rows r0 + 8 * (m >> 1), columns c0 + 8 * (m & 1)
__device__ __forceinline__ const bf16* at_cr(const bf16* p, int ld, int r0, int c0) {
  const int l = threadIdx.x & 31, m = l >> 3;
  return p + (r0 + (m >> 1) * 8 + (l & 7)) * ld + c0 + (m & 1) * 8;
}
// B operands (k x n) of two neighbouring n tiles: from a tile stored [n][k] resp. [k][n].
__device__ __forceinline__ void b_from_nk(uint32_t (&r)[4], const bf16* p, int ld, int n0, int k0) { ldsm(r, at_cr(p, ld, n0, k0)); }
__device__ __forceinline__ void b_from_kn(uint32_t (&r)[4], const bf16* p, int ld, int k0, int n0) { ldsm_t(r, at_rc(p, ld, k0, n0)); }
// A operand (m x k): from a tile stored [m][k] resp. [k][m].
__device__ __forceinline__ void a_from_mk(uint32_t (&r)[4], const bf16* p, int ld, int m0, int k0) { ldsm(r, at_rc(p, ld, m0, k0)); }
__device__ __forceinline__ void a_from_km(uint32_t (&r)[4], const bf16* p, int ld, int k0, int m0) { ldsm_t(r, at_cr(p, ld, k0, m0)); }

// Two accumulator tiles (columns 16 kk .. 16 kk + 15) as the high and low A operand of k step kk.
__device__ __forceinline__ void split_a(const float (&c0)[4], const float (&c1)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  split2(c0[0], c0[1], hi[0], lo[0]);
  split2(c0[2], c0[3], hi[1], lo[1]);
  split2(c1[0], c1[1], hi[2], lo[2]);
  split2(c1[2], c1[3], hi[3], lo[3]);
}

// The same with the remainder of the second rounding as a third part: the fp32 values themselves, but for 2^-26.
__device__ __forceinline__ void split_a3(const float (&c0)[4], const float (&c1)[4], uint32_t (&hi)[4], uint32_t (&lo)[4], uint32_t (&rest)[4]) {
  split3(c0[0], c0[1], hi[0], lo[0], rest[0]);
  split3(c0[2], c0[3], hi[1], lo[1], rest[1]);
  split3(c1[0], c1[1], hi[2], lo[2], rest[2]);
  split3(c1[2], c1[3], hi[3], lo[3], rest[3]);
}

// A strictly lower 64 x 64 matrix in two tiles, high and low parts: the blocks of 16 x 16 above the diagonal are never read
// as such, and hold what is left of the values, those of block (i, j) below the diagonal at (j, i) of the high parts' tile,
// those of the diagonal ones in the low parts' tile. Returns the place of block (i, j), i >= j.
__device__ __forceinline__ int rest_block(int i, int j) {
  return i > j ? 16 * j * APITCH + 16 * i : C * APITCH + (i < 3 ? 16 * (i + 1) : 16 * APITCH + 32);
}

// acc[2 * NT] += (hi + lo) x B for 2 * NT column tiles: one pass over all of them, then the other, so that no product
// waits for the one before it.
template <int NT>
__device__ __forceinline__ void mma2(float (*acc)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], const uint32_t (&b)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    mma(acc[2 * j], hi, b[j][0], b[j][1]);
    mma(acc[2 * j + 1], hi, b[j][2], b[j][3]);
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    mma(acc[2 * j], lo, b[j][0], b[j][1]);
    mma(acc[2 * j + 1], lo, b[j][2], b[j][3]);
  }
}

// ---------------------------------------------------------------------------------------------------- sequence plan

// cu <- running maximum of the given boundaries clamped to [0, T] (the boundaries themselves when they are valid, else
// the status word is set), cbase <- first chunk of every sequence. One block.
__global__ void plan_kernel(const int* __restrict__ in, int N, long long T, int* __restrict__ cu, int* __restrict__ cbase, int* status) {
  __shared__ int wmax[32], wsum[32], carry_max, carry_sum;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) carry_max = carry_sum = 0;
  __syncthreads();
  for (int base = 0; base <= N; base += blockDim.x) {
    const int i = base + tid;
    int x = 0;
    if (i <= N) {
      const int raw = in[i];
      x = raw < 0 ? 0 : (raw > T ? static_cast<int>(T) : raw);
      if (x != raw || (i > 0 && raw < in[i - 1])) *status = 7;
    }
    int m = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o && y > m) m = y;
    }
    if (lane == 31) wmax[warp] = m;
    __syncthreads();
    int top = carry_max;
    for (int w = 0; w < warp; ++w) top = wmax[w] > top ? wmax[w] : top;
    m = m > top ? m : top;
    if (i <= N) cu[i] = m;
    __syncthreads();
    if (tid == blockDim.x - 1) carry_max = m;
    __syncthreads();
  }
  __threadfence_block();
  __syncthreads();
  for (int base = 0; base <= N; base += blockDim.x) {
    const int i = base + tid;
    const int n = i < N ? (cu[i + 1] - cu[i] + C - 1) / C : 0;
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    if (lane == 31) wsum[warp] = s;
    __syncthreads();
    int before = carry_sum;
    for (int w = 0; w < warp; ++w) before += wsum[w];
    if (i <= N) cbase[i] = before + s - n;
    __syncthreads();
    if (tid == blockDim.x - 1) carry_sum = before + s;
    __syncthreads();
  }
}

// Zeroes the rows that no sequence covers, [0, cu[0]) and [cu[N], T), of a row-major buffer. The kernels that run anyway do
// it with their first blocks, whatever the device: a launch of its own costs a small call as much as its largest kernel.
constexpr int ZERO_BLOCKS = 128;
__device__ __forceinline__ void zero_rows(const DeltaArgs& a, long long first, long long last, void* buffer, long long words) {
  const long long n = (first + a.T - last) * words, step = static_cast<long long>(gridDim.x < ZERO_BLOCKS ? gridDim.x : ZERO_BLOCKS) * blockDim.x;
  for (long long w = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; w < n; w += step) {
    const long long r = w / words;
    static_cast<uint32_t*>(buffer)[(r < first ? r : last + (r - first)) * words + w % words] = 0u;
  }
}

// Copies a [64, cols] bf16 tile; rows from `len` on are zero.
template <int COLS, int THREADS>
__device__ __forceinline__ void load_rows(bf16* dst, int pitch, const bf16* src, long long stride, int len) {
  constexpr int V = COLS / 8;
  for (int i = threadIdx.x; i < C * V; i += THREADS) {
    const int r = i / V, v = i - r * V;
    const bool ok = r < len;
    cp16(dst + r * pitch + v * 8, src + (ok ? r * stride : 0) + v * 8, ok);
  }
}

// ---------------------------------------------------------------------------------------------------------- prepare

// 147 KB come and leave for each (chunk, key head) of 128 with two value heads: 92 us at 16384 tokens and 16 key heads,
// where the kernel takes 132 (4.6 TB/s). What is left is latency between the eight barriers of a head; four blocks of four
// warps share an SM (a fifth spills). The joins of the inverse on the matrix unit: 177 -> 132 us; records that leave by bulk
// copies instead of from the accumulators' owners, 16 bytes a row: 237 -> 177.

constexpr int PREP_THREADS = 128;
// fp32 pitches of the 64 x 64 matrices: A's is read down its columns as well (two rows 8 banks apart), M's along rows
constexpr int MP = 68, MMP = 72;

// Operands of fp32 matrices in shared memory, each value as a high and a low bf16 (16 bits of it), and the product of
// two such: what is left out is the low times the low.
struct Split2 { uint32_t hi[4], lo[4]; };
__device__ __forceinline__ void operand_a(Split2& o, const float* x, int pitch, int lane) {  // x [16 m, 16 k]
  const float* p = x + (lane >> 2) * pitch + (lane & 3) * 2;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v = *reinterpret_cast<const float2*>(p + (e & 1) * 8 * pitch + (e >> 1) * 8);
    split2(v.x, v.y, o.hi[e], o.lo[e]);
  }
}
__device__ __forceinline__ void operand_at(Split2& o, const float* x, int pitch, int lane) {  // x [16 k, 16 m]
  const float* p = x + (lane & 3) * 2 * pitch + (lane >> 2);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float* y = p + (e & 1) * 8 + (e >> 1) * 8 * pitch;
    split2(y[0], y[pitch], o.hi[e], o.lo[e]);
  }
}
__device__ __forceinline__ void mma_split(float (&d)[4], const Split2& x, const uint32_t (&hi)[2], const uint32_t (&lo)[2]) {
  mma(d, x.hi, hi[0], hi[1]);
  mma(d, x.hi, lo[0], lo[1]);
  mma(d, x.lo, hi[0], hi[1]);
}

// out = -Y (M X) for 16 columns of X and 16 rows of Y, KX and KY steps of 16 along the inner sides. (M X)^T comes out of
// the matrix unit as Y's second operand has to lie.
template <int KX, int KY>
__device__ __forceinline__ void join(float* out, const float* Y, const float* M, const float* X, int lane) {
  float m[2 * KY][4];
#pragma unroll
  for (int j = 0; j < 2 * KY; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) m[j][e] = 0.f;
#pragma unroll
  for (int k = 0; k < KX; ++k) {
    Split2 x;
    operand_at(x, X + 16 * k * MP, MP, lane);
#pragma unroll
    for (int j = 0; j < 2 * KY; ++j) {
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 v = *reinterpret_cast<const float2*>(M + (8 * j + (lane >> 2)) * MMP + 16 * k + 8 * e + (lane & 3) * 2);
        split2(v.x, v.y, hi[e], lo[e]);
      }
      mma_split(m[j], x, hi, lo);
    }
  }
  float s[2][4];
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
  for (int k = 0; k < KY; ++k) {
    Split2 y;
    operand_a(y, Y + 16 * k, MP, lane);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) split2(m[2 * k + e][2 * n], m[2 * k + e][2 * n + 1], hi[e], lo[e]);
      mma_split(s[n], y, hi, lo);
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(out + ((lane >> 2) + 8 * e) * MP + 8 * n + (lane & 3) * 2) =
          make_float2(-s[n][2 * e], -s[n][2 * e + 1]);
}

constexpr size_t PREP_PART = 2 * C * APITCH * sizeof(bf16);  // high and low of A, or of P, as they lie in the record
constexpr size_t PREP_TILES = 2 * PREP_PART + C * MP * sizeof(float);

// A contiguous piece of shared memory to device memory, behind a fence and a barrier of those who wrote it.
__device__ __forceinline__ void bulk_out(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_addr(src)), "r"(bytes)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// What this thread wrote to shared memory is seen by bulk copies that begin behind the next barrier.
__device__ __forceinline__ void fence_bulk() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bulk_out_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

template <int DK>
__global__ void __launch_bounds__(PREP_THREADS, 4)
prepare_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int P = DK + 8;
  bf16* qs = reinterpret_cast<bf16*>(smem);
  bf16* ks = qs + C * P;
  // q and k are in registers when these are written; M is done with when A is split into its place
  float* M = reinterpret_cast<float*>(smem);
  bf16* As = reinterpret_cast<bf16*>(smem);
  bf16* Ps = As + 2 * C * APITCH;
  float* A = reinterpret_cast<float*>(Ps + 2 * C * APITCH);
  float* rq = reinterpret_cast<float*>(smem + PREP_TILES);
  float* rk = rq + C;
  float* ghi = rk + C;
  float* glo = ghi + C;
  float* bt = glo + C;
  const long long c = blockIdx.x / a.Hk;
  const int hk = blockIdx.x % a.Hk;
  const Span sp = chunk_span(a, c);
  if (a.cu && blockIdx.x < ZERO_BLOCKS) zero_rows(a, a.cu[0], a.cu[a.N], a.o, a.Hv * a.dv / 2);
  if (sp.len == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  load_rows<DK, PREP_THREADS>(qs, P, static_cast<const bf16*>(a.q) + sp.start * a.q_ts + hk * a.q_hs, a.q_ts, sp.len);
  load_rows<DK, PREP_THREADS>(ks, P, static_cast<const bf16*>(a.k) + sp.start * a.k_ts + hk * a.k_hs, a.k_ts, sp.len);
  // the padding travels too, as zeros
  *reinterpret_cast<uint4*>(qs + tid * P + DK) = make_uint4(0, 0, 0, 0);
  cp_commit();
  cp_wait<0>();
  fence_bulk();
  __syncthreads();
  // the padded tiles as they are, for the kernels along the sequence: one bulk copy each there. k lies behind q.
  if (tid == 0) bulk_out(static_cast<bf16*>(a.qk) + (c * a.Hk + hk) * 2 * C * P, qs, 2 * C * P * sizeof(bf16));
  {
    const bf16* row = (tid < C ? qs : ks) + (tid & 63) * P;
    float ss = 0.f;
#pragma unroll 4
    for (int i = 0; i < DK / 8; ++i) {
      const uint4 w = reinterpret_cast<const uint4*>(row)[i];
      ss += lo_half(w.x) * lo_half(w.x) + hi_half(w.x) * hi_half(w.x);
      ss += lo_half(w.y) * lo_half(w.y) + hi_half(w.y) * hi_half(w.y);
      ss += lo_half(w.z) * lo_half(w.z) + hi_half(w.z) * hi_half(w.z);
      ss += lo_half(w.w) * lo_half(w.w) + hi_half(w.w) * hi_half(w.w);
    }
    (tid < C ? rq : rk)[tid & 63] = a.l2norm ? rsqrtf(ss + 1e-6f) : 1.f;
  }
  float kk[8][4], qk[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) kk[j][e] = qk[j][e] = 0.f;
#pragma unroll
  for (int s = 0; s < DK / 16; ++s) {
    uint32_t fq[4], fk[4], b[4];
    a_from_mk(fq, qs, P, warp * 16, s * 16);
    a_from_mk(fk, ks, P, warp * 16, s * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > warp) continue;  // columns behind the diagonal block
      b_from_nk(b, ks, P, j * 16, s * 16);
      mma(kk[2 * j], fk, b[0], b[1]);
      mma(kk[2 * j + 1], fk, b[2], b[3]);
      mma(qk[2 * j], fq, b[0], b[1]);
      mma(qk[2 * j + 1], fq, b[2], b[3]);
    }
  }
  const int rep = a.Hv / a.Hk;
  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    const long long rec = c * a.Hv + h;
    float* vec = a.vec + rec * DELTA_VEC;
    bf16* ap = static_cast<bf16*>(a.ap) + rec * DELTA_AP;
    if (tid == 0) bulk_out_read();  // what left from here is read
    __syncthreads();
    if (warp == 0) {
      // Running sum of g in 64 bits, kept as two floats: differences of neighbours stay exact next to strong decays.
      // Below -120 a decay is zero in fp32 whatever it is, and the sum stays finite.
      double s0 = 0.0, s1 = 0.0;
      const int i0 = 2 * lane, i1 = 2 * lane + 1;
      if (i0 < sp.len) { float x = a.g[(sp.start + i0) * a.Hv + h]; s0 = x < -120.f ? -120.f : x; }
      if (i1 < sp.len) { float x = a.g[(sp.start + i1) * a.Hv + h]; s1 = x < -120.f ? -120.f : x; }
      s1 += s0;
      double run = s1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += y;
      }
      const double before = run - s1;
      const double g0 = before + s0, g1 = run;
      ghi[i0] = static_cast<float>(g0);
      glo[i0] = static_cast<float>(g0 - static_cast<double>(ghi[i0]));
      ghi[i1] = static_cast<float>(g1);
      glo[i1] = static_cast<float>(g1 - static_cast<double>(ghi[i1]));
    } else if (warp >= 2) {
      // dbeta is (X . U) / beta: a beta of (nearly) zero becomes 1e-20, which writes nothing and still divides out
      const int i = tid - 64;
      float b = i < sp.len ? a.beta[(sp.start + i) * a.Hv + h] : 0.f;
      if (fabsf(b) < 1e-20f) b = b < 0.f ? -1e-20f : 1e-20f;
      bt[i] = b;
    }
    __syncthreads();
    if (tid < C) {
      const float gi = ghi[tid], gl = glo[tid], eg = __expf(gi) * (1.f + gl);
      vec[V_YK * 64 + tid] = rk[tid] * eg;
      vec[V_BETA * 64 + tid] = bt[tid];
      vec[V_OQ * 64 + tid] = a.scale * rq[tid] * eg;
      vec[V_SU * 64 + tid] = rk[tid] * __expf((ghi[63] - gi) + (glo[63] - gl));
      vec[V_GHI * 64 + tid] = gi;
      vec[V_GLO * 64 + tid] = gl;
      vec[V_QS * 64 + tid] = a.scale * rq[tid];
      vec[V_RK * 64 + tid] = rk[tid];
      vec[V_END * 64 + tid] = __expf(ghi[63]) * (1.f + glo[63]);
      vec[V_RQ * 64 + tid] = rq[tid];
    }
    float gih[2], gil[2], fq[2], fk[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = warp * 16 + g + 8 * e;
      gih[e] = ghi[i]; gil[e] = glo[i];
      fq[e] = a.scale * rq[i]; fk[e] = bt[i] * rk[i];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int j0 = 8 * j + t2;
      const float2 gh = *reinterpret_cast<const float2*>(ghi + j0), gl = *reinterpret_cast<const float2*>(glo + j0);
      const float2 rkj = *reinterpret_cast<const float2*>(rk + j0);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = warp * 16 + g + 8 * e;
        float m[2], p[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          // made everywhere and then selected: a branch per element costs its latency each time
          const int jj = j0 + f;
          const float d = (f ? rkj.y : rkj.x) * __expf((gih[e] - (f ? gh.y : gh.x)) + (gil[e] - (f ? gl.y : gl.x)));
          const float pv = fq[e] * d * qk[j][2 * e + f], mv = fk[e] * d * kk[j][2 * e + f];
          m[f] = i > jj ? mv : 0.f;
          p[f] = i > jj ? pv : 0.f;
          if (i == jj) vec[V_PD * 64 + i] = pv;
        }
        *reinterpret_cast<float2*>(M + i * MMP + j0) = make_float2(m[0], m[1]);
        if ((j >> 1) <= warp) {  // the block holds or meets the diagonal
          uint32_t hi, lo, rest;
          split3(p[0], p[1], hi, lo, rest);
          *reinterpret_cast<uint32_t*>(Ps + i * APITCH + j0) = hi;
          *reinterpret_cast<uint32_t*>(Ps + C * APITCH + i * APITCH + j0) = lo;
          *reinterpret_cast<uint32_t*>(Ps + rest_block(warp, j >> 1) + (i & 15) * APITCH + (j0 & 15)) = rest;
        }
      }
    }
    *reinterpret_cast<uint4*>(Ps + tid * APITCH + C) = make_uint4(0, 0, 0, 0);
    fence_bulk();
    __syncthreads();
    if (tid == 0) bulk_out(ap + 2 * C * APITCH, Ps, PREP_PART);
    // Inverse of I + M in fp32: the four 16 x 16 diagonal blocks by forward substitution, a thread per column ...
    if (tid < 64) {
      const int b0 = tid & 48, col = tid & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == col ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; j += 4) {
          const float4 m = *reinterpret_cast<const float4*>(M + (b0 + i) * MMP + b0 + j);
          s -= m.x * x[j];
          if (j + 1 < i) s -= m.y * x[j + 1];
          if (j + 2 < i) s -= m.z * x[j + 2];
          if (j + 3 < i) s -= m.w * x[j + 3];
        }
        x[i] = s;
        A[(b0 + i) * MP + b0 + col] = s;
      }
    }
    __syncthreads();
    // ... then [[X, 0], [M, Y]]^-1 has -Y^-1 M X^-1 below, for the two pairs of 16 and for the pair of 32, whose X^-1
    // and Y^-1 are lower triangular.
    if (warp < 2) {
      const int b0 = warp * 32;
      join<1, 1>(A + (b0 + 16) * MP + b0, A + (b0 + 16) * MP + b0 + 16, M + (b0 + 16) * MMP + b0, A + b0 * MP + b0, lane);
    }
    __syncthreads();
    if (warp == 0) join<2, 1>(A + 32 * MP, A + 32 * MP + 32, M + 32 * MMP, A, lane);
    if (warp == 1) join<2, 2>(A + 48 * MP, A + 48 * MP + 32, M + 32 * MMP, A, lane);
    if (warp == 2) join<1, 1>(A + 32 * MP + 16, A + 32 * MP + 32, M + 32 * MMP + 16, A + 16 * MP + 16, lane);
    if (warp == 3) join<1, 2>(A + 48 * MP + 16, A + 48 * MP + 32, M + 32 * MMP + 16, A + 16 * MP + 16, lane);
    __syncthreads();
    for (int w = tid; w < C * 8; w += PREP_THREADS) {
      const int r = w >> 3, c8 = (w & 7) * 8;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const bool below = (c8 >> 4) <= (r >> 4);
        float2 v = below ? *reinterpret_cast<const float2*>(A + r * MP + c8 + 2 * x) : make_float2(0.f, 0.f);
        if (r == c8 + 2 * x) v.x = 0.f;
        if (r == c8 + 2 * x + 1) v.y = 0.f;
        split2(v.x, v.y, hi[x], lo[x]);
      }
      *reinterpret_cast<uint4*>(As + r * APITCH + c8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(As + C * APITCH + r * APITCH + c8) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    *reinterpret_cast<uint4*>(As + tid * APITCH + C) = make_uint4(0, 0, 0, 0);
    fence_bulk();
    __syncthreads();
    if (tid == 0) bulk_out(ap, As, PREP_PART);
  }
  if (tid == 0) bulk_out_read();
}

template <int THREADS>
__device__ __forceinline__ void load_vec(float* dst, const float* src, int rows) {
  for (int i = threadIdx.x; i < rows * 16; i += THREADS) cp16(dst + i * 4, src + i * 4, true);
}

// ------------------------------------------------------------------------------------------- along the sequence: parts

// A unit is 16 columns of dv of one head and four warps. Warp w holds columns [w dk/4, (w + 1) dk/4) of the unit's state
// S^T [16, dk] in fp32, and makes everything that is per token for tokens [16 w, 16 w + 16) of a chunk. What the others
// need of it (the state, R, U) goes through shared memory as ready A operands, two or three parts, 16 bytes a lane each.
struct Operands {  // one k step of 16
  uint4 hi[32], lo[32];
};
__device__ __forceinline__ void put(Operands& x, const uint32_t (&hi)[4], const uint32_t (&lo)[4]) {
  const int lane = threadIdx.x & 31;
  x.hi[lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  x.lo[lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}
struct Operands3 {
  uint4 hi[32], lo[32], rest[32];
};
__device__ __forceinline__ void put(Operands3& x, const uint32_t (&hi)[4], const uint32_t (&lo)[4], const uint32_t (&rest)[4]) {
  const int lane = threadIdx.x & 31;
  x.hi[lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  x.lo[lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  x.rest[lane] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
}
__device__ __forceinline__ void get(const Operands3& x, uint32_t (&hi)[4], uint32_t (&lo)[4], uint32_t (&rest)[4]) {
  const int lane = threadIdx.x & 31;
  const uint4 h = x.hi[lane], l = x.lo[lane], r = x.rest[lane];
  hi[0] = h.x; hi[1] = h.y; hi[2] = h.z; hi[3] = h.w;
  lo[0] = l.x; lo[1] = l.y; lo[2] = l.z; lo[3] = l.w;
  rest[0] = r.x; rest[1] = r.y; rest[2] = r.z; rest[3] = r.w;
}
__device__ __forceinline__ void get(const Operands& x, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  const int lane = threadIdx.x & 31;
  const uint4 h = x.hi[lane], l = x.lo[lane];
  hi[0] = h.x; hi[1] = h.y; hi[2] = h.z; hi[3] = h.w;
  lo[0] = l.x; lo[1] = l.y; lo[2] = l.z; lo[3] = l.w;
}

// The calling thread's cp.async copies so far arrive on the barrier when they have landed.
__device__ __forceinline__ void bar_arrive_copies(uint64_t* b) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
// One thread copies a contiguous piece (16-byte aligned, a multiple of 16 bytes); it arrives on the barrier by its bytes.
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* b) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(b)) : "memory");
}

// Copies 64 rows x COLS bf16 (rows from `len` on become zeros), a 16-byte piece per thread.
template <int COLS, int THREADS>
__device__ __forceinline__ void copy_rows(bf16* dst, int pitch, const bf16* src, long long stride, int len) {
  constexpr int V = COLS / 8;
  static_assert(THREADS == C * V, "one piece a thread");
  const int r = threadIdx.x / V, v = (threadIdx.x % V) * 8;
  cp16(dst + r * pitch + v, src + (r < len ? r * stride : 0) + v, r < len);
}

// The warp's 16 tokens x 16 columns of fp32 accumulators, rounded to bf16, to rows of a token-major tensor through the
// warp's own `stage` [16][24].
constexpr int OUT_PITCH = 24;
__device__ __forceinline__ void store_tile(bf16* stage, bf16* out, long long stride, int len, const float (&c0)[4], const float (&c1)[4]) {
  const uint32_t r[4] = {pack2(c0[0], c0[1]), pack2(c0[2], c0[3]), pack2(c1[0], c1[1]), pack2(c1[2], c1[3])};
  __syncwarp();
  stsm_t(const_cast<bf16*>(at_cr(stage, OUT_PITCH, 0, 0)), r);
  __syncwarp();
  const int lane = threadIdx.x & 31, row = lane >> 1, v = (lane & 1) * 8;
  if (row < len) *reinterpret_cast<uint4*>(out + row * stride + v) = *reinterpret_cast<const uint4*>(stage + row * OUT_PITCH + v);
}
// The fp32 values of a fragment's three parts.
__device__ __forceinline__ void join(const uint32_t (&hi)[4], const uint32_t (&lo)[4], const uint32_t (&rest)[4], float (&c)[2][4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i >> 1][2 * (i & 1)] = lo_half(hi[i]) + (lo_half(lo[i]) + lo_half(rest[i]));
    c[i >> 1][2 * (i & 1) + 1] = hi_half(hi[i]) + (hi_half(lo[i]) + hi_half(rest[i]));
  }
}
// Accumulators as they are kept for the backward pass, and back.
__device__ __forceinline__ void keep(uint4* dst, const float (&c)[2][4]) {
#pragma unroll
  for (int f = 0; f < 2; ++f)
    dst[32 * f] = make_uint4(__float_as_uint(c[f][0]), __float_as_uint(c[f][1]), __float_as_uint(c[f][2]), __float_as_uint(c[f][3]));
}
__device__ __forceinline__ void kept(const uint4 (&x)[2], float (&c)[2][4]) {
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    c[f][0] = __uint_as_float(x[f].x);
    c[f][1] = __uint_as_float(x[f].y);
    c[f][2] = __uint_as_float(x[f].z);
    c[f][3] = __uint_as_float(x[f].w);
  }
}

// Values of a factor row for the lane's four tokens: tile f, element pair.
__device__ __forceinline__ void factors(const float* row, float2 (&x)[2]) {
  x[0] = *reinterpret_cast<const float2*>(row);
  x[1] = *reinterpret_cast<const float2*>(row + 8);
}
// c[f][e] *= x for the token of element e
__device__ __forceinline__ void scale_tokens(float (&c)[2][4], const float2 (&x)[2]) {
#pragma unroll
  for (int f = 0; f < 2; ++f) {
    c[f][0] *= x[f].x;
    c[f][1] *= x[f].y;
    c[f][2] *= x[f].x;
    c[f][3] *= x[f].y;
  }
}
__device__ __forceinline__ void clear(float (&c)[2][4]) {
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[f][e] = 0.f;
}
__device__ __forceinline__ void mma_pair(float (&c)[2][4], const uint32_t (&a)[4], const uint32_t (&b)[4]) {
  mma(c[0], a, b[0], b[1]);
  mma(c[1], a, b[2], b[3]);
}
__device__ __forceinline__ void add_to(float (&c)[2][4], const float (&d)[2][4]) {
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[f][e] += d[f][e];
}

// ---------------------------------------------------------------------------------------------------------- forward

template <int DK, int NU>
struct FwdStage {
  static constexpr int P = DK + DELTA_ROW_PAD, VP = NU * 16 + 8;
  bf16 qk[2 * C * P], ap[DELTA_AP], v[C * VP];
  float vec[SEQ_ROWS * 64];
  static constexpr uint32_t BULK = (2 * C * P + DELTA_AP) * sizeof(bf16) + SEQ_ROWS * 64 * sizeof(float);
};
template <int DK, int NU>
struct FwdSmem {
  FwdStage<DK, NU> stage[2];
  Operands state[NU][DK / 16];
  Operands3 r[NU][4], u[NU][4], su[NU][4];
  bf16 out[NU * 4][16 * OUT_PITCH];
  uint64_t full[2], empty[2], state_ready[NU], r_ready[NU], u_ready[NU];
};

// KEEP: also write what the backward pass needs; the results are the same, bit by bit.
template <int DK, int NU, bool KEEP>
__global__ void __launch_bounds__(NU * 128, 1)
forward_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Smem = FwdSmem<DK, NU>;
  using Stage = FwdStage<DK, NU>;
  constexpr int P = Stage::P, VP = Stage::VP, THREADS = NU * 128, KT = DK / 16, KW = KT / 4;
  Smem& sm = *reinterpret_cast<Smem*>(smem);
  const int splits = a.dv / (NU * 16);
  const int vb = blockIdx.x % splits, h = (blockIdx.x / splits) % a.Hv, n = blockIdx.x / (splits * a.Hv);
  const int hk = h / (a.Hv / a.Hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, unit = warp >> 2, w = warp & 3, g = lane >> 2, t2 = (lane & 3) * 2;
  const int col0 = vb * NU * 16 + unit * 16;  // the unit's first column of dv
  const long long start = a.cu ? a.cu[n] : 0, end = a.cu ? a.cu[n + 1] : a.T, c0 = a.cu ? a.cbase[n] : 0;
  const int chunks = static_cast<int>((end - start + C - 1) / C);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(&sm.full[i], THREADS + 1);
      bar_init(&sm.empty[i], NU * 4);
    }
    for (int i = 0; i < NU; ++i) {
      bar_init(&sm.state_ready[i], 4);
      bar_init(&sm.r_ready[i], 4);
      bar_init(&sm.u_ready[i], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  float s[2 * KW][4];  // rows = columns of dv, columns = dk [16 KW w, 16 KW (w + 1))
  const long long sbase = (static_cast<long long>(n) * a.Hv + h) * DK * a.dv + col0;
  const int kd0 = 16 * KW * w;
#pragma unroll
  for (int j = 0; j < 2 * KW; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[j][e] = a.s_in ? a.s_in[sbase + static_cast<long long>(kd0 + 8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] : 0.f;

  auto fetch = [&](int c) {
    Stage& x = sm.stage[c & 1];
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const long long rec = (c0 + c) * a.Hv + h;
    copy_rows<NU * 16, THREADS>(x.v, VP, static_cast<const bf16*>(a.v) + t0 * a.v_ts + h * a.v_hs + vb * NU * 16, a.v_ts, len);
    bar_arrive_copies(&sm.full[c & 1]);
    if (threadIdx.x == 0) {
      bar_expect(&sm.full[c & 1], Stage::BULK);
      bulk_copy(x.qk, static_cast<const bf16*>(a.qk) + ((c0 + c) * a.Hk + hk) * 2 * C * P, sizeof(x.qk), &sm.full[c & 1]);
      bulk_copy(x.ap, static_cast<const bf16*>(a.ap) + rec * DELTA_AP, sizeof(x.ap), &sm.full[c & 1]);
      bulk_copy(x.vec, a.vec + rec * DELTA_VEC, sizeof(x.vec), &sm.full[c & 1]);
    }
  };
  // The state in front of the next chunk: for the unit's other warps, and (keep_state) for the backward pass.
  uint32_t ph[KW][4], pl[KW][4];
  auto publish_state = [&]() {
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      split_a(s[2 * k], s[2 * k + 1], ph[k], pl[k]);
      put(sm.state[unit][KW * w + k], ph[k], pl[k]);
    }
    bar_arrive(&sm.state_ready[unit]);
  };
  auto keep_state = [&](int c) {
    uint4* sf = reinterpret_cast<uint4*>(a.states) + ((((c0 + c) * a.Hv + h) * (a.dv / 16) + (col0 >> 4)) * 2) * KT * 32 + lane;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      sf[(KW * w + k) * 32] = make_uint4(ph[k][0], ph[k][1], ph[k][2], ph[k][3]);
      sf[(KT + KW * w + k) * 32] = make_uint4(pl[k][0], pl[k][1], pl[k][2], pl[k][3]);
    }
  };
  if (chunks > 0) {
    fetch(0);
    publish_state();
    if (KEEP) keep_state(0);
  }
  for (int c = 0; c < chunks; ++c) {
    Stage& x = sm.stage[c & 1];
    const uint32_t parity = c & 1, turn = (c >> 1) & 1;
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const bf16 *xq = x.qk, *xk = x.qk + C * P, *ahi = x.ap, *alo = x.ap + C * APITCH, *phi = x.ap + 2 * C * APITCH, *plo = x.ap + 3 * C * APITCH;
    const int tok = 16 * w;  // the warp's first token
    const float* vec = x.vec + tok + t2;
    if (c + 1 < chunks) {  // the other buffer is free when all warps are done with chunk c - 1
      if (c > 0) bar_wait(&sm.empty[(c + 1) & 1], ((c - 1) >> 1) & 1, a.status);
      fetch(c + 1);
    }
    bar_wait(&sm.full[c & 1], turn, a.status);
    // everything that does not wait for the state is in registers before it comes
    uint32_t bk[KT][4], v[4];
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) b_from_nk(bk[kk], xk, P, tok, 16 * kk);
    a_from_km(v, x.v, VP, tok, unit * 16);
    float2 yk[2], be[2];
    factors(vec + V_YK * 64, yk);
    factors(vec + V_BETA * 64, be);
    bar_wait(&sm.state_ready[unit], parity, a.status);

    // (K S)^T of the warp's tokens
    float y[2][4], z[2][4];
    uint32_t sh[KT][4], sl[KT][4];
    clear(y);
    clear(z);
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) get(sm.state[unit][kk], sh[kk], sl[kk]);
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      mma_pair(y, sh[kk], bk[kk]);
      mma_pair(z, sl[kk], bk[kk]);
    }
    add_to(y, z);
    // r = beta (V - e^G K S)^T
    scale_tokens(y, yk);
    float u[2][4];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      u[f][0] = be[f].x * (lo_half(v[2 * f]) - y[f][0]);
      u[f][1] = be[f].y * (hi_half(v[2 * f]) - y[f][1]);
      u[f][2] = be[f].x * (lo_half(v[2 * f + 1]) - y[f][2]);
      u[f][3] = be[f].y * (hi_half(v[2 * f + 1]) - y[f][3]);
    }
    uint32_t rh[4], rl[4], rr[4];  // the warp's own part of r
    split_a3(u[0], u[1], rh, rl, rr);
    put(sm.r[unit][w], rh, rl, rr);
    bar_arrive(&sm.r_ready[unit]);
    // while the others get there: (A - I) r with the warp's own part, the rest of A, and e^G Q S. The output is made for
    // tokens [tok2, tok2 + 16), mirrored: the warp with the most of A has the least of P.
    const int tok2 = 48 - tok;
    const float* vec2 = x.vec + tok2 + t2;
    uint32_t ab[3][2][4];
#pragma unroll
    for (int kk = 0; kk < 3; ++kk)
      if (kk < w) {
        b_from_nk(ab[kk][0], ahi, APITCH, tok, 16 * kk);
        b_from_nk(ab[kk][1], alo, APITCH, tok, 16 * kk);
      }
    float m[2][4], m2[2][4], m3[2][4];
    clear(m);
    clear(m2);
    clear(m3);
    {
      uint32_t b[4], bl[4];
      b_from_nk(b, ahi, APITCH, tok, tok);
      b_from_nk(bl, alo, APITCH, tok, tok);
      mma_pair(m, rh, b);
      mma_pair(m2, rl, b);
      mma_pair(m3, rh, bl);
      mma_pair(m2, rr, b);
      mma_pair(m3, rl, bl);
    }
    float2 f2[2], ib[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) ib[f] = make_float2(__fdividef(1.f, be[f].x), __fdividef(1.f, be[f].y));
    factors(vec + V_SU * 64, f2);
    bar_wait(&sm.r_ready[unit], parity, a.status);
    // (A - I) r; the memory read at each token is m = e^G K S - ((A - I) r) / beta, and U = beta (V - m), which enters its
    // products in three parts: what they and the sums of dg see of U must be the same to fp32.
#pragma unroll
    for (int kk = 0; kk < 3; ++kk)
      if (kk < w) {
        uint32_t hi[4], lo[4], rest[4];
        get(sm.r[unit][kk], hi, lo, rest);
        mma_pair(m, hi, ab[kk][0]);
        mma_pair(m2, lo, ab[kk][0]);
        mma_pair(m3, hi, ab[kk][1]);
        mma_pair(m2, rest, ab[kk][0]);
        mma_pair(m3, lo, ab[kk][1]);
      }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      m[f][0] = y[f][0] - (m[f][0] + (m2[f][0] + m3[f][0])) * ib[f].x;
      m[f][1] = y[f][1] - (m[f][1] + (m2[f][1] + m3[f][1])) * ib[f].y;
      m[f][2] = y[f][2] - (m[f][2] + (m2[f][2] + m3[f][2])) * ib[f].x;
      m[f][3] = y[f][3] - (m[f][3] + (m2[f][3] + m3[f][3])) * ib[f].y;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u[i >> 1][2 * (i & 1)] = be[i >> 1].x * (lo_half(v[i]) - m[i >> 1][2 * (i & 1)]);
      u[i >> 1][2 * (i & 1) + 1] = be[i >> 1].y * (hi_half(v[i]) - m[i >> 1][2 * (i & 1) + 1]);
    }
    {
      float su[2][4];
      uint32_t hi[4], lo[4], rest[4];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) su[f][e] = u[f][e];
      scale_tokens(su, f2);
      split_a3(su[0], su[1], hi, lo, rest);
      put(sm.su[unit][w], hi, lo, rest);
      split_a3(u[0], u[1], hi, lo, rest);
      put(sm.u[unit][w], hi, lo, rest);
    }
    bar_arrive(&sm.u_ready[unit]);
    // meanwhile: K for the state, e^G Q S, and what is kept
    const float ge = x.vec[V_END * 64];
#pragma unroll
    for (int j = 0; j < 2 * KW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] *= ge;
    uint32_t bt[4][KW][4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int j = 0; j < KW; ++j) b_from_kn(bt[kk][j], xk, P, 16 * kk, kd0 + 16 * j);
    float o[2][4];
    clear(o);
    clear(z);
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      uint32_t b[4];
      b_from_nk(b, xq, P, tok2, 16 * kk);
      mma_pair(o, sh[kk], b);
      mma_pair(z, sl[kk], b);
    }
    bar_wait(&sm.u_ready[unit], parity, a.status);
    // S^T <- e^{G_C} S^T + (e^{G_C - G} U)^T K, the warp's columns of dk
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4], rest[4];
      get(sm.su[unit][kk], hi, lo, rest);
      mma2<KW>(s, hi, lo, bt[kk]);
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        mma(s[2 * j], rest, bt[kk][j][0], bt[kk][j][1]);
        mma(s[2 * j + 1], rest, bt[kk][j][2], bt[kk][j][3]);
      }
    }
    if (c + 1 < chunks) publish_state();
    // what earlier tokens give to the output: + (P - diag P) U, but for what is below 2^-26 of it: the backward pass
    // multiplies with this P too
    add_to(o, z);
    factors(vec2 + V_OQ * 64, f2);
    scale_tokens(o, f2);
    clear(z);
    clear(m2);
    clear(m3);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      if (kk <= 3 - w) {
        uint32_t hi[4], lo[4], rest[4], b[4], bl[4];
        b_from_nk(b, phi, APITCH, tok2, 16 * kk);
        b_from_nk(bl, plo, APITCH, tok2, 16 * kk);
        get(sm.u[unit][kk], hi, lo, rest);
        mma_pair(o, hi, b);
        mma_pair(z, lo, b);
        mma_pair(m2, hi, bl);
        mma_pair(m3, lo, bl);
        mma_pair(m3, rest, b);
        b_from_nk(b, phi + rest_block(3 - w, kk), APITCH, 0, 0);
        mma_pair(m2, hi, b);
      }
    add_to(m2, m3);
    add_to(z, m2);
    add_to(o, z);
    if (KEEP) {
      const long long piece = (((c0 + c) * a.Hv + h) * (a.dv / 16) + (col0 >> 4)) * 4;
      keep(reinterpret_cast<uint4*>(a.mem) + (piece + w) * 64 + lane, m);
      keep(reinterpret_cast<uint4*>(a.u) + (piece + w) * 64 + lane, u);
      keep(reinterpret_cast<uint4*>(a.past) + (piece + 3 - w) * 64 + lane, o);
      if (c + 1 < chunks) keep_state(c + 1);
    }
    {
      uint32_t hi[4], lo[4], rest[4];
      get(sm.u[unit][3 - w], hi, lo, rest);
      join(hi, lo, rest, u);
    }
    factors(vec2 + V_PD * 64, f2);
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      o[f][0] += f2[f].x * u[f][0];
      o[f][1] += f2[f].y * u[f][1];
      o[f][2] += f2[f].x * u[f][2];
      o[f][3] += f2[f].y * u[f][3];
    }
    bar_arrive(&sm.empty[c & 1]);
    store_tile(sm.out[warp], static_cast<bf16*>(a.o) + ((t0 + tok2) * a.Hv + h) * a.dv + col0, static_cast<long long>(a.Hv) * a.dv,
               len - tok2, o[0], o[1]);
  }
  if (a.s_out) {
#pragma unroll
    for (int j = 0; j < 2 * KW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        a.s_out[sbase + static_cast<long long>(kd0 + 8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] = s[j][e];
  }
}

// --------------------------------------------------------------------------------------------------------- backward

template <int DK, int NU>
struct BwdStage {
  static constexpr int P = DK + DELTA_ROW_PAD, VP = NU * 16 + 8;
  bf16 qk[2 * C * P], ap[DELTA_AP], dO[C * VP];
  float vec[SEQ_ROWS * 64];
  static constexpr uint32_t BULK = (2 * C * P + DELTA_AP) * sizeof(bf16) + SEQ_ROWS * 64 * sizeof(float);
};
template <int DK, int NU>
struct BwdSmem {
  BwdStage<DK, NU> stage[2];
  Operands state[NU][DK / 16], dv[NU][4], go[NU][4];
  Operands3 du[NU][4];
  bf16 out[NU * 4][16 * OUT_PITCH];
  uint64_t full[2], empty[2], state_ready[NU], du_ready[NU], dv_ready[NU];
};

template <int DK, int NU>
__global__ void __launch_bounds__(NU * 128, 1)
backward_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Smem = BwdSmem<DK, NU>;
  using Stage = BwdStage<DK, NU>;
  constexpr int P = Stage::P, VP = Stage::VP, THREADS = NU * 128, KT = DK / 16, KW = KT / 4;
  Smem& sm = *reinterpret_cast<Smem*>(smem);
  const int splits = a.dv / (NU * 16);
  const int vb = blockIdx.x % splits, h = (blockIdx.x / splits) % a.Hv, n = blockIdx.x / (splits * a.Hv);
  const int hk = h / (a.Hv / a.Hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, unit = warp >> 2, w = warp & 3, g = lane >> 2, t2 = (lane & 3) * 2;
  const int col0 = vb * NU * 16 + unit * 16, VT = a.dv / 16, vt = col0 >> 4;
  const long long start = a.cu ? a.cu[n] : 0, end = a.cu ? a.cu[n + 1] : a.T, c0 = a.cu ? a.cbase[n] : 0;
  const int chunks = static_cast<int>((end - start + C - 1) / C);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(&sm.full[i], THREADS + 1);
      bar_init(&sm.empty[i], NU * 4);
    }
    for (int i = 0; i < NU; ++i) {
      bar_init(&sm.state_ready[i], 4);
      bar_init(&sm.du_ready[i], 4);
      bar_init(&sm.dv_ready[i], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  float s[2 * KW][4];  // dS^T, the warp's columns of dk
  const long long sbase = (static_cast<long long>(n) * a.Hv + h) * DK * a.dv + col0;
  const int kd0 = 16 * KW * w;
#pragma unroll
  for (int j = 0; j < 2 * KW; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[j][e] = a.ds_out ? a.ds_out[sbase + static_cast<long long>(kd0 + 8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] : 0.f;

  // i counts the chunks from the last one
  auto fetch = [&](int i) {
    Stage& x = sm.stage[i & 1];
    const int c = chunks - 1 - i;
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const long long rec = (c0 + c) * a.Hv + h;
    const long long row = (t0 * a.Hv + h) * a.dv + vb * NU * 16, stride = static_cast<long long>(a.Hv) * a.dv;
    copy_rows<NU * 16, THREADS>(x.dO, VP, static_cast<const bf16*>(a.dout) + row, stride, len);
    bar_arrive_copies(&sm.full[i & 1]);
    if (threadIdx.x == 0) {
      bar_expect(&sm.full[i & 1], Stage::BULK);
      bulk_copy(x.qk, static_cast<const bf16*>(a.qk) + ((c0 + c) * a.Hk + hk) * 2 * C * P, sizeof(x.qk), &sm.full[i & 1]);
      bulk_copy(x.ap, static_cast<const bf16*>(a.ap) + rec * DELTA_AP, sizeof(x.ap), &sm.full[i & 1]);
      bulk_copy(x.vec, a.vec + rec * DELTA_VEC, sizeof(x.vec), &sm.full[i & 1]);
    }
  };
  // The gradient of the state behind a chunk: for the unit's other warps, and (keep_state) for dqk.
  uint32_t ph[KW][4], pl[KW][4];
  auto publish_state = [&]() {
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      split_a(s[2 * k], s[2 * k + 1], ph[k], pl[k]);
      put(sm.state[unit][KW * w + k], ph[k], pl[k]);
    }
    bar_arrive(&sm.state_ready[unit]);
  };
  auto keep_state = [&](int c) {
    uint4* df = reinterpret_cast<uint4*>(a.dstates) + (((c0 + c) * a.Hv + h) * VT + vt) * 2 * KT * 32 + lane;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      df[(KW * w + k) * 32] = make_uint4(ph[k][0], ph[k][1], ph[k][2], ph[k][3]);
      df[(KT + KW * w + k) * 32] = make_uint4(pl[k][0], pl[k][1], pl[k][2], pl[k][3]);
    }
  };
  // What a chunk's warp reads of the forward pass: its part of the state in front, and m, U, past of its tokens.
  struct Kept {
    uint4 sh[KW], sl[KW], m[2], u[2], past[2];
  } now, next;
  auto load_kept = [&](int c, Kept& x) {
    const long long piece = ((c0 + c) * a.Hv + h) * VT + vt;
    const uint4* nf = reinterpret_cast<const uint4*>(a.states) + piece * 2 * KT * 32 + lane;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      x.sh[k] = nf[(KW * w + k) * 32];
      x.sl[k] = nf[(KT + KW * w + k) * 32];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      x.m[k] = (reinterpret_cast<const uint4*>(a.mem) + (piece * 4 + w) * 64 + lane)[32 * k];
      x.u[k] = (reinterpret_cast<const uint4*>(a.u) + (piece * 4 + w) * 64 + lane)[32 * k];
      x.past[k] = (reinterpret_cast<const uint4*>(a.past) + (piece * 4 + w) * 64 + lane)[32 * k];
    }
  };
  if (chunks > 0) {
    fetch(0);
    load_kept(chunks - 1, next);
    publish_state();
    keep_state(chunks - 1);
  }
  for (int i = 0; i < chunks; ++i) {
    const int c = chunks - 1 - i;
    Stage& x = sm.stage[i & 1];
    const uint32_t parity = i & 1, turn = (i >> 1) & 1;
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const long long rec = (c0 + c) * a.Hv + h;
    const bf16 *xq = x.qk, *xk = x.qk + C * P, *ahi = x.ap, *alo = x.ap + C * APITCH, *phi = x.ap + 2 * C * APITCH, *plo = x.ap + 3 * C * APITCH;
    const int tok = 16 * w;
    const float* vec = x.vec + tok + t2;
    now = next;
    if (i + 1 < chunks) {
      load_kept(c - 1, next);
      if (i > 0) bar_wait(&sm.empty[(i + 1) & 1], ((i - 1) >> 1) & 1, a.status);
      fetch(i + 1);
    }
    bar_wait(&sm.full[i & 1], turn, a.status);

    // what does not wait for the state: ((P - diag P)^T dO)^T of the warp's tokens, K and factors
    float u[2][4], z[2][4], y[2][4], du[2][4];
    clear(u);
    clear(z);
    uint32_t fo[4];  // dO^T of the warp's tokens
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      if (kk >= w) {
        uint32_t f[4], b[4], bl[4];
        a_from_km(f, x.dO, VP, 16 * kk, unit * 16);
        b_from_kn(b, phi, APITCH, 16 * kk, tok);
        b_from_kn(bl, plo, APITCH, 16 * kk, tok);
        mma_pair(u, f, b);
        mma_pair(z, f, bl);
        b_from_kn(b, phi + rest_block(kk, w), APITCH, 0, 0);
        mma_pair(z, f, b);
      }
    a_from_km(fo, x.dO, VP, tok, unit * 16);
    float2 f2[2], su[2], be[2];
    factors(vec + V_OQ * 64, f2);
    uint32_t gh[4], gl[4];  // e^G dO, for the state
#pragma unroll
    for (int e = 0; e < 4; ++e) split2(lo_half(fo[e]) * f2[e >> 1].x, hi_half(fo[e]) * f2[e >> 1].y, gh[e], gl[e]);
    add_to(u, z);
    factors(vec + V_PD * 64, f2);
#pragma unroll
    for (int f = 0; f < 2; ++f) {  // diag P dO
      du[f][0] = f2[f].x * lo_half(fo[2 * f]);
      du[f][1] = f2[f].y * hi_half(fo[2 * f]);
      du[f][2] = f2[f].x * lo_half(fo[2 * f + 1]);
      du[f][3] = f2[f].y * hi_half(fo[2 * f + 1]);
    }
    factors(vec + V_SU * 64, su);
    uint32_t bk[KT][4];
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) b_from_nk(bk[kk], xk, P, tok, 16 * kk);
    bar_wait(&sm.state_ready[unit], parity, a.status);
    put(sm.go[unit][w], gh, gl);  // not before: the last chunk's is read until the state is published
    // y = (e^{G_C - G} K dS1)^T
    clear(y);
    clear(z);
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      uint32_t hi[4], lo[4];
      get(sm.state[unit][kk], hi, lo);
      mma_pair(y, hi, bk[kk]);
      mma_pair(z, lo, bk[kk]);
    }
    add_to(y, z);
    scale_tokens(y, su);
    // dU^T = y + u + (diag P dO)^T
    add_to(u, y);
    uint32_t dh[4], dl[4], dr[4];
    {
      float d[2][4];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) d[f][e] = u[f][e] + du[f][e];
      split_a3(d[0], d[1], dh, dl, dr);
      put(sm.du[unit][w], dh, dl, dr);
    }
    bar_arrive(&sm.du_ready[unit]);
    // while the others get there: U + dU^T (A - I) begins with the warp's own part
    const float ge = x.vec[V_END * 64];
    float mm[2][4], uu[2][4];
    kept(now.m, mm);
    kept(now.u, uu);
    float sdot = 0.f, bdot = 0.f;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) bdot += y[f][e] * uu[f][e];
    uint32_t ab[3][2][4];
#pragma unroll
    for (int kk = 1; kk < 4; ++kk)
      if (kk > w) {
        b_from_kn(ab[kk - 1][0], ahi, APITCH, 16 * kk, tok);
        b_from_kn(ab[kk - 1][1], alo, APITCH, 16 * kk, tok);
      }
    clear(y);
    clear(z);
    {
      uint32_t b[4], bl[4];
      b_from_kn(b, ahi, APITCH, tok, tok);
      b_from_kn(bl, alo, APITCH, tok, tok);
      mma_pair(u, dh, b);
      mma_pair(y, dl, b);
      mma_pair(z, dh, bl);
      mma_pair(y, dr, b);
      mma_pair(z, dl, bl);
    }
    factors(vec + V_BETA * 64, be);
    factors(vec + V_YK * 64, f2);
    bar_wait(&sm.du_ready[unit], parity, a.status);
    // u <- u + dU^T (A - I): X without what the token's own output asks for
#pragma unroll
    for (int kk = 1; kk < 4; ++kk)
      if (kk > w) {
        uint32_t hi[4], lo[4], rest[4];
        get(sm.du[unit][kk], hi, lo, rest);
        mma_pair(u, hi, ab[kk - 1][0]);
        mma_pair(y, lo, ab[kk - 1][0]);
        mma_pair(z, hi, ab[kk - 1][1]);
        mma_pair(y, rest, ab[kk - 1][0]);
        mma_pair(z, lo, ab[kk - 1][1]);
      }
    add_to(y, z);
    add_to(u, y);
    // X = u + (diag P dO)^T, dV = beta X; row sums over the unit's 16 columns: past . dO - m . dV - U . u, U . X and U . dO
    float d[ROW_DOTS][4];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      d[0][2 * f] = -(uu[f][0] * u[f][0] + uu[f][2] * u[f][2]);
      d[0][2 * f + 1] = -(uu[f][1] * u[f][1] + uu[f][3] * u[f][3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[f][e] += du[f][e];
      d[1][2 * f] = uu[f][0] * u[f][0] + uu[f][2] * u[f][2];
      d[1][2 * f + 1] = uu[f][1] * u[f][1] + uu[f][3] * u[f][3];
    }
    scale_tokens(u, be);
    {
      float b[2][4];
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[f][e] = -u[f][e];
      scale_tokens(b, f2);
      split_a(b[0], b[1], hi, lo);
      put(sm.dv[unit][w], hi, lo);
    }
    bar_arrive(&sm.dv_ready[unit]);
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const float* past = reinterpret_cast<const float*>(&now.past[f]);
      d[2][2 * f] = uu[f][0] * lo_half(fo[2 * f]) + uu[f][2] * lo_half(fo[2 * f + 1]);
      d[2][2 * f + 1] = uu[f][1] * hi_half(fo[2 * f]) + uu[f][3] * hi_half(fo[2 * f + 1]);
      d[0][2 * f] += past[0] * lo_half(fo[2 * f]) + past[2] * lo_half(fo[2 * f + 1]) - (mm[f][0] * u[f][0] + mm[f][2] * u[f][2]);
      d[0][2 * f + 1] += past[1] * hi_half(fo[2 * f]) + past[3] * hi_half(fo[2 * f + 1]) - (mm[f][1] * u[f][1] + mm[f][3] * u[f][3]);
    }
    // while the others get there: <dS1, S0>, and Q^T diag(e^G) dO into the state
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const uint32_t wh[4] = {now.sh[k].x, now.sh[k].y, now.sh[k].z, now.sh[k].w}, wl[4] = {now.sl[k].x, now.sl[k].y, now.sl[k].z, now.sl[k].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sdot += s[2 * k + (e >> 1)][2 * (e & 1)] * (lo_half(wh[e]) + lo_half(wl[e]));
        sdot += s[2 * k + (e >> 1)][2 * (e & 1) + 1] * (hi_half(wh[e]) + hi_half(wl[e]));
      }
    }
    sdot = sdot * ge + bdot;
#pragma unroll
    for (int j = 0; j < 2 * KW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] *= ge;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4], b[KW][4];
#pragma unroll
      for (int j = 0; j < KW; ++j) b_from_kn(b[j], xq, P, 16 * kk, kd0 + 16 * j);
      get(sm.go[unit][kk], hi, lo);
      mma2<KW>(s, hi, lo, b);
    }
    uint32_t bt[4][KW][4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int j = 0; j < KW; ++j) b_from_kn(bt[kk][j], xk, P, 16 * kk, kd0 + 16 * j);
    bar_wait(&sm.dv_ready[unit], parity, a.status);
    // dS0 -= K^T diag(e^G) dV
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4];
      get(sm.dv[unit][kk], hi, lo);
      mma2<KW>(s, hi, lo, bt[kk]);
    }
    if (c > 0) publish_state();
    bar_arrive(&sm.empty[i & 1]);
    if (c > 0) keep_state(c - 1);
    store_tile(sm.out[warp], static_cast<bf16*>(a.dv_) + ((t0 + tok) * a.Hv + h) * a.dv + col0,
               static_cast<long long>(a.Hv) * a.dv, len - tok, u[0], u[1]);
    {  // what that rounding left of dV, for dqk
      uint32_t hi[4], lo[4];
      split_a(u[0], u[1], hi, lo);
      reinterpret_cast<uint4*>(a.dv_lo)[((rec * VT + vt) * 4 + w) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    float* rd = a.rowdots + (rec * VT + vt) * ROW_DOTS * 64 + tok + t2;
#pragma unroll
    for (int q = 0; q < ROW_DOTS; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float r = d[q][e];
        r += __shfl_xor_sync(0xffffffffu, r, 4);
        r += __shfl_xor_sync(0xffffffffu, r, 8);
        r += __shfl_xor_sync(0xffffffffu, r, 16);
        if (g == 0) rd[q * 64 + 8 * (e >> 1) + (e & 1)] = r;
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sdot += __shfl_xor_sync(0xffffffffu, sdot, o);
    if (lane == 0) a.sdots[(rec * VT + vt) * 4 + w] = sdot;
  }
  if (a.ds_in) {
#pragma unroll
    for (int j = 0; j < 2 * KW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        a.ds_in[sbase + static_cast<long long>(kd0 + 8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] = s[j][e];
  }
}

// -------------------------------------------------------------------------------------------------------------- dqk

template <int DK, int DV>
struct DqkSmem {
  static constexpr int P = DK + 8, VP = DV + 8;
  // names in l: what the rounding to bf16 left
  bf16 q[C * P], k[C * P], dO[C * VP], dV[C * VP], dVl[DV * APITCH], u[DV * APITCH], ul[DV * APITCH];
  bf16 s0[DV * P], s0l[DV * P], ds[DV * P], dsl[DV * P];
  bf16 w1[C * APITCH], w1l[C * APITCH], w2[C * APITCH], w2l[C * APITCH];
  float vec[8 * 64];
  float dots[2][2][C];
};

constexpr int DQK_THREADS = 256;

// State fragments of all dv / 16 column tiles, high and low parts -> [DV][DK] rows of pitch DK + 8.
template <int DK, int DV>
__device__ __forceinline__ void load_fragments(bf16* hi, bf16* lo, const uint4* src) {
  constexpr int KT = DK / 16, P = DK + 8;
  for (int i = threadIdx.x; i < DV / 16 * 2 * KT * 32; i += DQK_THREADS) {
    const int lane = i & 31, kk = (i >> 5) % KT, part = (i >> 5) / KT & 1, vt = (i >> 5) / (2 * KT), g = lane >> 2, t2 = (lane & 3) * 2;
    const uint4 f = src[i];
    bf16* p = (part ? lo : hi) + (vt * 16 + g) * P + kk * 16 + t2;
    *reinterpret_cast<uint32_t*>(p) = f.x;
    *reinterpret_cast<uint32_t*>(p + 8 * P) = f.y;
    *reinterpret_cast<uint32_t*>(p + 8) = f.z;
    *reinterpret_cast<uint32_t*>(p + 8 * P + 8) = f.w;
  }
}

// A fragment of 16 columns and 16 tokens to [DV][64 tokens] rows of pitch APITCH.
__device__ __forceinline__ void put_tokens(bf16* tile, int vt, int w, int lane, const uint32_t (&f)[4]) {
  bf16* p = tile + (vt * 16 + (lane >> 2)) * APITCH + w * 16 + (lane & 3) * 2;
  *reinterpret_cast<uint32_t*>(p) = f[0];
  *reinterpret_cast<uint32_t*>(p + 8 * APITCH) = f[1];
  *reinterpret_cast<uint32_t*>(p + 8) = f[2];
  *reinterpret_cast<uint32_t*>(p + 8 * APITCH + 8) = f[3];
}
// U^T, kept in fp32, in its two parts; and what the rounding of dV^T left.
template <int DV>
__device__ __forceinline__ void load_tokens(bf16* uh, bf16* ul, bf16* dvl, const uint4* u, const uint4* v) {
  for (int i = threadIdx.x; i < DV / 16 * 128; i += DQK_THREADS) {
    const int lane = i & 31, w = (i >> 5) & 3, vt = i >> 7;
    const uint4 x[2] = {u[(i >> 5) * 64 + lane], u[(i >> 5) * 64 + 32 + lane]}, y = v[i];
    float c[2][4];
    kept(x, c);
    uint32_t hi[4], lo[4];
    split_a(c[0], c[1], hi, lo);
    put_tokens(uh, vt, w, lane, hi);
    put_tokens(ul, vt, w, lane, lo);
    const uint32_t d[4] = {y.x, y.y, y.z, y.w};
    put_tokens(dvl, vt, w, lane, d);
  }
}

template <int DK, int DV>
__global__ void __launch_bounds__(DQK_THREADS, 1)
dqk_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Smem = DqkSmem<DK, DV>;
  Smem& x = *reinterpret_cast<Smem*>(smem);
  constexpr int P = Smem::P, VP = Smem::VP, KT = DK / 16, NT = DK / 16;  // NT: 8-wide column tiles of a half of dk
  const long long c = blockIdx.x / a.Hk;
  const int hk = blockIdx.x % a.Hk, rep = a.Hv / a.Hk;
  const Span sp = chunk_span(a, c);
  if (sp.len == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wm = warp & 3, wn = warp >> 2, g = lane >> 2, t2 = (lane & 3) * 2;
  const int r0 = wm * 16 + g, n0 = wn * (DK / 2);
  load_rows<DK, DQK_THREADS>(x.q, P, static_cast<const bf16*>(a.q) + sp.start * a.q_ts + hk * a.q_hs, a.q_ts, sp.len);
  load_rows<DK, DQK_THREADS>(x.k, P, static_cast<const bf16*>(a.k) + sp.start * a.k_ts + hk * a.k_hs, a.k_ts, sp.len);
  float dq[NT][4], dk[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) dq[j][e] = dk[j][e] = 0.f;
  float wd[2] = {0.f, 0.f};  // diagonal of W in the thread's rows
  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    const long long rec = c * a.Hv + h;
    const long long row = (sp.start * a.Hv + h) * a.dv, stride = static_cast<long long>(a.Hv) * a.dv;
    __syncthreads();
    load_rows<DV, DQK_THREADS>(x.dO, VP, static_cast<const bf16*>(a.dout) + row, stride, sp.len);
    load_rows<DV, DQK_THREADS>(x.dV, VP, static_cast<const bf16*>(a.dv_) + row, stride, sp.len);
    load_vec<DQK_THREADS>(x.vec, a.vec + rec * DELTA_VEC, 8);
    cp_commit();
    load_tokens<DV>(x.u, x.ul, x.dVl, reinterpret_cast<const uint4*>(a.u) + rec * (DV / 16) * 256,
                    reinterpret_cast<const uint4*>(a.dv_lo) + rec * (DV / 16) * 128);
    load_fragments<DK, DV>(x.s0, x.s0l, reinterpret_cast<const uint4*>(a.states) + rec * (DV / 16) * 2 * KT * 32);
    load_fragments<DK, DV>(x.ds, x.dsl, reinterpret_cast<const uint4*>(a.dstates) + rec * (DV / 16) * 2 * KT * 32);
    cp_wait<0>();
    __syncthreads();
    // dO U^T and dV U^T, 16 x 32 of each per warp, lower part only
    float p[4][4], nn[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) p[j][e] = nn[j][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DV / 16; ++kk) {
      uint32_t fo[4], fv[4], fvl[4], b[4], bl[4];
      a_from_mk(fo, x.dO, VP, wm * 16, kk * 16);
      a_from_mk(fv, x.dV, VP, wm * 16, kk * 16);
      a_from_km(fvl, x.dVl, APITCH, kk * 16, wm * 16);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (wn * 2 + j > wm) continue;
        b_from_kn(b, x.u, APITCH, kk * 16, wn * 32 + j * 16);
        mma(p[2 * j], fo, b[0], b[1]);
        mma(p[2 * j + 1], fo, b[2], b[3]);
        mma(nn[2 * j], fv, b[0], b[1]);
        mma(nn[2 * j + 1], fv, b[2], b[3]);
        b_from_kn(bl, x.ul, APITCH, kk * 16, wn * 32 + j * 16);
        mma(p[2 * j], fo, bl[0], bl[1]);
        mma(p[2 * j + 1], fo, bl[2], bl[3]);
        mma(nn[2 * j], fv, bl[0], bl[1]);
        mma(nn[2 * j + 1], fv, bl[2], bl[3]);
        mma(nn[2 * j], fvl, b[0], b[1]);
        mma(nn[2 * j + 1], fvl, b[2], b[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (wn * 2 + (j >> 1) > wm) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = r0 + 8 * (e >> 1), jj = wn * 32 + j * 8 + t2 + (e & 1);
        float w1 = 0.f, w2 = 0.f;
        if (i > jj) {
          const float d = x.vec[V_RK * 64 + jj] * __expf((x.vec[V_GHI * 64 + i] - x.vec[V_GHI * 64 + jj]) + (x.vec[V_GLO * 64 + i] - x.vec[V_GLO * 64 + jj]));
          w1 = x.vec[V_QS * 64 + i] * d * p[j][e];
          w2 = -x.vec[V_RK * 64 + i] * d * nn[j][e];
        }
        const bf16 w1h = __float2bfloat16(w1);
        x.w1[i * APITCH + jj] = w1h;
        x.w1l[i * APITCH + jj] = __float2bfloat16(w1 - __bfloat162float(w1h));
        if (i >= jj) {  // N + N^T
          const bf16 w2h = __float2bfloat16(w2), w2r = __float2bfloat16(w2 - __bfloat162float(w2h));
          x.w2[i * APITCH + jj] = x.w2[jj * APITCH + i] = w2h;
          x.w2l[i * APITCH + jj] = x.w2l[jj * APITCH + i] = w2r;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) wd[e] += w_diagonal(a, rec, r0 + 8 * e, x.vec);
    // the products with the states: rows scaled afterwards
    float t[NT][4];
    auto clear = [&]() {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[j][e] = 0.f;
    };
    auto product = [&](const bf16* rows, const bf16* state, bool transposed) {
#pragma unroll
      for (int kk = 0; kk < DV / 16; ++kk) {
        uint32_t f[4], b[4];
        if (transposed) a_from_km(f, rows, APITCH, kk * 16, wm * 16); else a_from_mk(f, rows, VP, wm * 16, kk * 16);
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
          b_from_kn(b, state, P, kk * 16, n0 + j * 16);
          mma(t[2 * j], f, b[0], b[1]);
          mma(t[2 * j + 1], f, b[2], b[3]);
        }
      }
    };
    auto add = [&](float(&acc)[NT][4], float f0, float f1) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        acc[j][0] += f0 * t[j][0];
        acc[j][1] += f0 * t[j][1];
        acc[j][2] += f1 * t[j][2];
        acc[j][3] += f1 * t[j][3];
      }
    };
    clear();
    product(x.dO, x.s0, false);
    product(x.dO, x.s0l, false);
    add(dq, x.vec[V_OQ * 64 + r0], x.vec[V_OQ * 64 + r0 + 8]);
    clear();
    product(x.dV, x.s0, false);
    product(x.dV, x.s0l, false);
    product(x.dVl, x.s0, true);
    add(dk, -x.vec[V_YK * 64 + r0], -x.vec[V_YK * 64 + r0 + 8]);
    clear();
    product(x.u, x.ds, true);
    product(x.u, x.dsl, true);
    product(x.ul, x.ds, true);
    add(dk, x.vec[V_SU * 64 + r0], x.vec[V_SU * 64 + r0 + 8]);
    __syncthreads();  // w1, w2
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t f1[4], f1l[4], ft[4], ftl[4], f2[4], f2l[4], b[4];
      a_from_mk(f1, x.w1, APITCH, wm * 16, kk * 16);
      a_from_mk(f1l, x.w1l, APITCH, wm * 16, kk * 16);
      a_from_km(ft, x.w1, APITCH, kk * 16, wm * 16);
      a_from_km(ftl, x.w1l, APITCH, kk * 16, wm * 16);
      a_from_mk(f2, x.w2, APITCH, wm * 16, kk * 16);
      a_from_mk(f2l, x.w2l, APITCH, wm * 16, kk * 16);
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        b_from_kn(b, x.k, P, kk * 16, n0 + j * 16);
        if (kk <= wm) {
          mma(dq[2 * j], f1, b[0], b[1]);
          mma(dq[2 * j + 1], f1, b[2], b[3]);
          mma(dq[2 * j], f1l, b[0], b[1]);
          mma(dq[2 * j + 1], f1l, b[2], b[3]);
        }
        mma(dk[2 * j], f2, b[0], b[1]);
        mma(dk[2 * j + 1], f2, b[2], b[3]);
        mma(dk[2 * j], f2l, b[0], b[1]);
        mma(dk[2 * j + 1], f2l, b[2], b[3]);
        if (kk >= wm) {
          b_from_kn(b, x.q, P, kk * 16, n0 + j * 16);
          mma(dk[2 * j], ft, b[0], b[1]);
          mma(dk[2 * j + 1], ft, b[2], b[3]);
          mma(dk[2 * j], ftl, b[0], b[1]);
          mma(dk[2 * j + 1], ftl, b[2], b[3]);
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = (r0 + 8 * e) * P + n0 + 8 * j + t2;
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(x.k + at), qw = *reinterpret_cast<const uint32_t*>(x.q + at);
      dq[j][2 * e] += wd[e] * lo_half(kw);
      dq[j][2 * e + 1] += wd[e] * hi_half(kw);
      dk[j][2 * e] += wd[e] * lo_half(qw);
      dk[j][2 * e + 1] += wd[e] * hi_half(qw);
    }
  // The accumulators hold r dq^ and r dk^ with r = 1 / norm, so that dq = r dq^ - q r^2 (q . r dq^), the same for k.
  auto finish = [&](float(&acc)[NT][4], bf16* tile, int which, const float* r) {
    if (a.l2norm) {
      float d0 = 0.f, d1 = 0.f;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t x0 = *reinterpret_cast<const uint32_t*>(tile + r0 * P + n0 + 8 * j + t2);
        const uint32_t x1 = *reinterpret_cast<const uint32_t*>(tile + (r0 + 8) * P + n0 + 8 * j + t2);
        d0 += acc[j][0] * lo_half(x0) + acc[j][1] * hi_half(x0);
        d1 += acc[j][2] * lo_half(x1) + acc[j][3] * hi_half(x1);
      }
      d0 += __shfl_xor_sync(0xffffffffu, d0, 1);
      d0 += __shfl_xor_sync(0xffffffffu, d0, 2);
      d1 += __shfl_xor_sync(0xffffffffu, d1, 1);
      d1 += __shfl_xor_sync(0xffffffffu, d1, 2);
      if ((lane & 3) == 0) {
        x.dots[which][wn][r0] = d0;
        x.dots[which][wn][r0 + 8] = d1;
      }
    }
    __syncthreads();
    float f0 = 0.f, f1 = 0.f;
    if (a.l2norm) {
      f0 = (x.dots[which][0][r0] + x.dots[which][1][r0]) * r[r0] * r[r0];
      f1 = (x.dots[which][0][r0 + 8] + x.dots[which][1][r0 + 8]) * r[r0 + 8] * r[r0 + 8];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {  // every element is read and replaced by the same thread
      uint32_t* p0 = reinterpret_cast<uint32_t*>(tile + r0 * P + n0 + 8 * j + t2);
      uint32_t* p1 = reinterpret_cast<uint32_t*>(tile + (r0 + 8) * P + n0 + 8 * j + t2);
      *p0 = pack2(acc[j][0] - f0 * lo_half(*p0), acc[j][1] - f0 * hi_half(*p0));
      *p1 = pack2(acc[j][2] - f1 * lo_half(*p1), acc[j][3] - f1 * hi_half(*p1));
    }
  };
  const float* factors = a.vec + (c * a.Hv + hk * rep) * DELTA_VEC;
  finish(dq, x.q, 0, factors + V_RQ * 64);
  finish(dk, x.k, 1, factors + V_RK * 64);
  __syncthreads();
  constexpr int V = DK / 8;
  for (int i = threadIdx.x; i < C * V; i += DQK_THREADS) {
    const int r = i / V, v = (i - r * V) * 8;
    if (r >= sp.len) continue;
    const long long o = ((sp.start + r) * a.Hk + hk) * DK + v;
    *reinterpret_cast<uint4*>(static_cast<bf16*>(a.dq) + o) = *reinterpret_cast<const uint4*>(x.q + r * P + v);
    *reinterpret_cast<uint4*>(static_cast<bf16*>(a.dkey) + o) = *reinterpret_cast<const uint4*>(x.k + r * P + v);
  }
}

// ------------------------------------------------------------------------------------------------------------ gates

// One warp per (chunk, value head): sums over the units, then dbeta and the suffix sums of dg in 64 bits.
constexpr int GATE_WARPS = 4;
__global__ void __launch_bounds__(GATE_WARPS * 32)
gates_kernel(const DeltaArgs a) {
  if (a.cu && blockIdx.x < ZERO_BLOCKS) {
    const long long first = a.cu[0], last = a.cu[a.N];
    zero_rows(a, first, last, a.dq, a.Hk * a.dk / 2);
    zero_rows(a, first, last, a.dkey, a.Hk * a.dk / 2);
    zero_rows(a, first, last, a.dv_, a.Hv * a.dv / 2);
    zero_rows(a, first, last, a.dg, a.Hv);
    zero_rows(a, first, last, a.dbeta, a.Hv);
  }
  const unsigned pair = blockIdx.x * GATE_WARPS + (threadIdx.x >> 5);  // at most 2^31 of them
  const int c = static_cast<int>(pair / static_cast<unsigned>(a.Hv)), h = static_cast<int>(pair - c * static_cast<unsigned>(a.Hv));
  const long long rec = pair;
  if (c >= a.NC) return;
  const Span sp = chunk_span(a, c);
  if (sp.len == 0) return;
  const int lane = threadIdx.x & 31, VT = a.dv / 16;
  const float* rd = a.rowdots + rec * VT * ROW_DOTS * 64;
  double carry = lane < 4 * VT ? a.sdots[rec * 4 * VT + lane] : 0.f;  // dv / 4 <= 32 of them
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) carry += __shfl_xor_sync(0xffffffffu, carry, o);
#pragma unroll
  for (int half = 1; half >= 0; --half) {
    const int i = half * 32 + lane;
    double s = 0.0, xu = 0.0;
    for (int v = 0; v < VT; ++v) {
      s += rd[v * ROW_DOTS * 64 + i];
      xu += rd[(v * ROW_DOTS + 1) * 64 + i];
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_down_sync(0xffffffffu, s, o);
      if (lane + o < 32) s += y;
    }
    s += carry;
    carry = __shfl_sync(0xffffffffu, s, 0);
    if (i < sp.len) {
      const long long at = (sp.start + i) * a.Hv + h;
      a.dg[at] = static_cast<float>(s);
      a.dbeta[at] = static_cast<float>(xu / a.vec[rec * DELTA_VEC + V_BETA * 64 + i]);
    }
  }
}

// --------------------------------------------------------------------------------------------------------- launches

template <int DK, int NU, bool KEEP>
int launch_forward(const DeltaArgs& a, cudaStream_t s) {
  const long long grid = static_cast<long long>(a.N) * a.Hv * (a.dv / (NU * 16));
  if (grid > INT32_MAX) return -2;
  const size_t bytes = sizeof(FwdSmem<DK, NU>);
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(forward_kernel<DK, NU, KEEP>, bytes, allowed)) return -3;
  forward_kernel<DK, NU, KEEP><<<static_cast<unsigned>(grid), NU * 128, bytes, s>>>(a);
  return 0;
}

template <int DK, int NU>
int launch_backward(const DeltaArgs& a, cudaStream_t s) {
  const long long grid = static_cast<long long>(a.N) * a.Hv * (a.dv / (NU * 16));
  if (grid > INT32_MAX) return -2;
  const size_t bytes = sizeof(BwdSmem<DK, NU>);
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(backward_kernel<DK, NU>, bytes, allowed)) return -3;
  backward_kernel<DK, NU><<<static_cast<unsigned>(grid), NU * 128, bytes, s>>>(a);
  return 0;
}

template <int DK, int DV>
int launch_dqk(const DeltaArgs& a, cudaStream_t s) {
  const size_t bytes = sizeof(DqkSmem<DK, DV>);
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(dqk_kernel<DK, DV>, bytes, allowed)) return -3;
  dqk_kernel<DK, DV><<<static_cast<unsigned>(a.NC * a.Hk), DQK_THREADS, bytes, s>>>(a);
  return 0;
}

template <int DK>
int forward_dk(const DeltaArgs& a, cudaStream_t s) {
  if (a.NC > 0) {
    const size_t bytes = PREP_TILES + 5 * C * sizeof(float);
    static std::atomic<uint64_t> allowed{0};
    if (!allow_smem(prepare_kernel<DK>, bytes, allowed)) return -3;
    prepare_kernel<DK><<<static_cast<unsigned>(a.NC * a.Hk), PREP_THREADS, bytes, s>>>(a);
  }
  const int rc = a.states ? launch_forward<DK, 2, true>(a, s) : launch_forward<DK, 2, false>(a, s);
  if (rc) return rc;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

template <int DK>
int backward_dk(const DeltaArgs& a, cudaStream_t s) {
  int rc = launch_backward<DK, 2>(a, s);
  if (rc) return rc;
  if (a.NC > 0) {
    if (a.dv == 64) rc = launch_dqk<DK, 64>(a, s);
    else if constexpr (DK == 128) rc = delta_tc_dqk(a, s);
    else rc = launch_dqk<DK, 128>(a, s);
    if (rc) return rc;
    gates_kernel<<<static_cast<unsigned>((a.NC * a.Hv + GATE_WARPS - 1) / GATE_WARPS), GATE_WARPS * 32, 0, s>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

bool covered(const DeltaArgs& a) {
  return (a.dk == 64 || a.dk == 128) && (a.dv == 64 || a.dv == 128) && a.Hk > 0 && a.Hv % a.Hk == 0 && a.NC * a.Hv <= INT32_MAX;
}

}  // namespace

int delta_plan(const int* cu_in, int N, long long T, int* cu, int* cbase, int* status, cudaStream_t s) {
  plan_kernel<<<1, 1024, 0, s>>>(cu_in, N, T, cu, cbase, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int delta_forward(const DeltaArgs& a, cudaStream_t s) {
  if (!covered(a)) return -1;
  return a.dk == 64 ? forward_dk<64>(a, s) : forward_dk<128>(a, s);
}

int delta_backward(const DeltaArgs& a, cudaStream_t s) {
  if (!covered(a)) return -1;
  return a.dk == 64 ? backward_dk<64>(a, s) : backward_dk<128>(a, s);
}

}  // namespace lf
