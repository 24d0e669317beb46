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
//   dQ = diag(e^G) dO S0^T + W K,   W = lower(dO U^T) D
//   dK = -diag(e^G) dV S0^T + diag(e^{G_C - G}) U dS1^T + W^T Q + (N + N^T) K,   N = -strict_lower(dV U^T) D
//
// The gradient of a log decay g_t gathers what every token or state in front of t gives to every token or state from t
// on. With o~_i the part of o_i, and m_i = v_i - u_i / beta_i the part of the memory read at i, that earlier tokens
// wrote, and x~_j the part of X_j that later tokens ask for,
//
//   dg_t = sum_{i >= t} (o~_i.do_i - m_i.dv_i) - sum_{j >= t} u_j.x~_j + sum_j e^{G_C - G_j} (K dS1)_j.u_j + e^{G_C} <dS1, S0>
//
// with sums over the chunk. Every term carries a decay, so strongly decaying heads keep the relative accuracy of their
// (small) gradient; that is why A and P are kept as strict lower parts, their diagonals apart: o~, m and x~ are sums of
// their own, never differences of larger numbers.
//
// Kernels:
//   prepare   one block per (chunk, key head): Q K^T and K K^T once, then A, P and the per-token factors of each of its
//             value heads.
//   forward   one warp owns 16 of the dv columns of a head and walks along the sequence; the delta rule acts on every
//             column by itself, so a warp never waits for another one. It keeps S^T [16, dk] in the accumulators of
//             mma.sync and works on transposed products throughout: an accumulator tile is then, register by register,
//             the A operand of the next product, and nothing of the chain S -> K S -> U -> S goes through shared memory.
//   backward  the same in reverse with dS^T.
//   dqk       one block per (chunk, key head): dQ and dK, parallel over chunks.
//   gates     dg and dbeta.
//
// Precision. The state, U, X and all products along the chain carry 16 or more bits: an fp32 operand is cut into a bf16
// high and low part (relative remainder 2^-18) and multiplied in two passes where the other operand is a bf16 input
// (q, k, do), in three where both are cut. That keeps states, dg and dbeta at fp32 accuracy. dQ and dK are only needed to
// bf16: there S0, dS1, dV and N enter with the high part alone (2^-9 relative each, in terms that decay has made small);
// U and W, whose products can cancel to little when keys are alike, keep both parts.
//
// The chain is bound by the tensor pipe's latency and rate at one warp per scheduler, not by bandwidth; mma.sync runs at
// a quarter of tcgen05's rate but its operands and results stay in registers.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "linear_attn.h"

namespace lf {
namespace {

using bf16 = __nv_bfloat16;
constexpr int C = DELTA_CHUNK;
constexpr int APITCH = 72;  // bf16 per row of a 64-wide tile: odd multiple of 16 bytes, no bank conflicts in ldmatrix

// ------------------------------------------------------------------------------------------------------- primitives

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

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
__device__ __forceinline__ void cp16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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

__device__ __forceinline__ uint32_t pack2(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float lo_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// x, y -> bf16 pair and the bf16 pair of what the rounding left. Volatile, so that the parts of a whole state are made
// again where they are used again instead of being held in registers in between.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
  lo = pack2(x - lo_half(hi), y - hi_half(hi));
}
// Two accumulator tiles (columns 16 kk .. 16 kk + 15) as the high and low A operand of k step kk.
__device__ __forceinline__ void split_a(const float (&c0)[4], const float (&c1)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  split2(c0[0], c0[1], hi[0], lo[0]);
  split2(c0[2], c0[3], hi[1], lo[1]);
  split2(c1[0], c1[1], hi[2], lo[2]);
  split2(c1[2], c1[3], hi[3], lo[3]);
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

struct Span {
  int n;            // sequence
  long long start;  // first token of the chunk
  int len;          // its tokens, 1 .. 64; 0 = no such chunk
};

__device__ __forceinline__ Span chunk_span(const DeltaArgs& a, long long c) {
  Span s;
  if (a.cu == nullptr) {
    s.n = 0;
    s.start = c * C;
    const long long left = a.T - s.start;
    s.len = left <= 0 ? 0 : (left < C ? static_cast<int>(left) : C);
    return s;
  }
  if (c >= a.cbase[a.N]) {
    s.n = 0;
    s.start = 0;
    s.len = 0;
    return s;
  }
  int lo = 0, hi = a.N;  // last n with cbase[n] <= c; sequences without tokens have no chunk and are passed over
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cbase[mid] <= c) lo = mid; else hi = mid;
  }
  s.n = lo;
  s.start = a.cu[lo] + (c - a.cbase[lo]) * C;
  const long long left = a.cu[lo + 1] - s.start;
  s.len = left < C ? static_cast<int>(left) : C;
  return s;
}

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

__global__ void zero_rows_kernel(const ZeroRows z, const int* __restrict__ cu, int N, long long T) {
  const long long first = cu[0], last = cu[N], rows = first + T - last;
  if (rows <= 0) return;
  for (int i = 0; i < z.n; ++i) {
    const long long words = z.row_bytes[i] / 4;
    uint32_t* p = static_cast<uint32_t*>(z.p[i]);
    for (long long w = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; w < rows * words; w += static_cast<long long>(gridDim.x) * blockDim.x) {
      const long long r = w / words;
      p[(r < first ? r : last + (r - first)) * words + w % words] = 0u;
    }
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

// Rows of a chunk's factor block, 64 floats each.
enum { V_YK = 0, V_BETA, V_OQ, V_SU, V_GHI, V_GLO, V_QS, V_RK, V_END, V_PD, V_RQ };  // V_PD: diagonal of P
constexpr int SEQ_ROWS = V_PD + 1;  // rows that the kernels along the sequence read

constexpr int PREP_THREADS = 128;
constexpr int MP = 68;  // fp32 pitch of the 64 x 64 matrices: rows 16-byte aligned, neighbours four banks apart

template <int DK>
__global__ void __launch_bounds__(PREP_THREADS)
prepare_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int P = DK + 8;
  bf16* qs = reinterpret_cast<bf16*>(smem);
  bf16* ks = qs + C * P;
  float* M = reinterpret_cast<float*>(ks + C * P);
  float* A = M + C * MP;
  float* rq = A + C * MP;
  float* rk = rq + C;
  float* ghi = rk + C;
  float* glo = ghi + C;
  float* bt = glo + C;
  const long long c = blockIdx.x / a.Hk;
  const int hk = blockIdx.x % a.Hk;
  const Span sp = chunk_span(a, c);
  if (sp.len == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  load_rows<DK, PREP_THREADS>(qs, P, static_cast<const bf16*>(a.q) + sp.start * a.q_ts + hk * a.q_hs, a.q_ts, sp.len);
  load_rows<DK, PREP_THREADS>(ks, P, static_cast<const bf16*>(a.k) + sp.start * a.k_ts + hk * a.k_hs, a.k_ts, sp.len);
  cp_commit();
  cp_wait<0>();
  __syncthreads();
  {
    const bf16* row = (tid < C ? qs : ks) + (tid & 63) * P;
    float ss = 0.f;
#pragma unroll 4
    for (int i = 0; i < DK / 2; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(row)[i];
      ss += lo_half(w) * lo_half(w) + hi_half(w) * hi_half(w);
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
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = warp * 16 + g + 8 * e, j0 = 8 * j + t2;
        float m[2], p[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int jj = j0 + f;
          m[f] = p[f] = 0.f;
          if (i >= jj) {
            const float d = rk[jj] * __expf((ghi[i] - ghi[jj]) + (glo[i] - glo[jj]));
            p[f] = a.scale * rq[i] * d * qk[j][2 * e + f];
            if (i > jj) {
              m[f] = bt[i] * rk[i] * d * kk[j][2 * e + f];
            } else {
              vec[V_PD * 64 + i] = p[f];
              p[f] = 0.f;
            }
          }
        }
        *reinterpret_cast<float2*>(M + i * MP + j0) = make_float2(m[0], m[1]);
        uint32_t hi, lo;
        split2(p[0], p[1], hi, lo);
        *reinterpret_cast<uint32_t*>(ap + 2 * C * C + i * C + j0) = hi;
        *reinterpret_cast<uint32_t*>(ap + 3 * C * C + i * C + j0) = lo;
      }
    }
    __syncthreads();
    // Inverse of I + M in fp32: the four 16 x 16 diagonal blocks by forward substitution, a thread per column ...
    if (tid < 64) {
      const int b0 = tid & 48, col = tid & 15;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float s = i == col ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i; ++j) s -= M[(b0 + i) * MP + b0 + j] * x[j];
        x[i] = s;
        A[(b0 + i) * MP + b0 + col] = s;
      }
    }
    __syncthreads();
    // ... then the blocks below, a diagonal at a time: A_IJ = -A_II sum_{J <= K < I} M_IK A_KJ. A thread makes four
    // neighbouring columns of one row.
    for (int d = 1; d < 4; ++d) {
      for (int w = tid; w < (4 - d) * 64; w += PREP_THREADS) {
        const int J = w >> 6, I = J + d, r = (w >> 2) & 15, cc = (w & 3) * 4;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int K = J * 16; K < I * 16; K += 4) {
          const float4 m = *reinterpret_cast<const float4*>(M + (I * 16 + r) * MP + K);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float mv = x == 0 ? m.x : x == 1 ? m.y : x == 2 ? m.z : m.w;
            const float4 v = *reinterpret_cast<const float4*>(A + (K + x) * MP + J * 16 + cc);
            s.x += mv * v.x; s.y += mv * v.y; s.z += mv * v.z; s.w += mv * v.w;
          }
        }
        // the sum goes where the result will lie; A_IJ is not read before the next diagonal
        *reinterpret_cast<float4*>(A + (I * 16 + r) * MP + J * 16 + cc) = s;
      }
      __syncthreads();
      float4 res[2];
      int n = 0;
      for (int w = tid; w < (4 - d) * 64; w += PREP_THREADS, ++n) {
        const int J = w >> 6, I = J + d, r = (w >> 2) & 15, cc = (w & 3) * 4;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float mv = A[(I * 16 + r) * MP + I * 16 + x];
          const float4 v = *reinterpret_cast<const float4*>(A + (I * 16 + x) * MP + J * 16 + cc);
          s.x -= mv * v.x; s.y -= mv * v.y; s.z -= mv * v.z; s.w -= mv * v.w;
        }
        if (n == 0) res[0] = s; else res[1] = s;
      }
      __syncthreads();
      n = 0;
      for (int w = tid; w < (4 - d) * 64; w += PREP_THREADS, ++n) {
        const int J = w >> 6, I = J + d, r = (w >> 2) & 15, cc = (w & 3) * 4;
        *reinterpret_cast<float4*>(A + (I * 16 + r) * MP + J * 16 + cc) = n == 0 ? res[0] : res[1];
      }
      __syncthreads();
    }
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
      *reinterpret_cast<uint4*>(ap + r * C + c8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(ap + C * C + r * C + c8) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- forward

template <int COLS, int THREADS>
__device__ __forceinline__ void load_square(bf16* dst, const bf16* src) {  // n x [64, 64] contiguous -> pitch APITCH
  for (int i = threadIdx.x; i < COLS * C * 8; i += THREADS) {
    const int r = i >> 3, v = i & 7;
    cp16(dst + r * APITCH + v * 8, src + r * C + v * 8, true);
  }
}

template <int THREADS>
__device__ __forceinline__ void load_vec(float* dst, const float* src, int rows) {
  for (int i = threadIdx.x; i < rows * 16; i += THREADS) cp16(dst + i * 4, src + i * 4, true);
}

// The warp's [16 columns, 64 tokens] tile of fp32 accumulators, rounded to bf16, to rows of a token-major tensor
// through `stage` (the warp's own columns of a [64, pitch] tile).
template <typename F>
__device__ __forceinline__ void store_tokens(bf16* stage, int pitch, bf16* out, long long stride, int len, F value) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    uint32_t r[4];
    r[0] = pack2(value(j, 0), value(j, 1));
    r[1] = pack2(value(j, 2), value(j, 3));
    r[2] = pack2(value(j + 1, 0), value(j + 1, 1));
    r[3] = pack2(value(j + 1, 2), value(j + 1, 3));
    stsm_t(const_cast<bf16*>(at_cr(stage, pitch, 8 * j, 0)), r);
  }
  __syncwarp();
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 16 + (lane >> 1), v = (lane & 1) * 8;
    if (r < len) *reinterpret_cast<uint4*>(out + r * stride + v) = *reinterpret_cast<const uint4*>(stage + r * pitch + v);
  }
  __syncwarp();
}

// Two neighbouring tokens of one column: m from its parts, U = beta (v - m).
__device__ __forceinline__ void memory_term(uint32_t v, uint32_t mh, uint32_t ml, float2 beta, float& m0, float& m1, float& u0, float& u1) {
  m0 = lo_half(mh) + lo_half(ml);
  m1 = hi_half(mh) + hi_half(ml);
  u0 = beta.x * (lo_half(v) - m0);
  u1 = beta.y * (hi_half(v) - m1);
}

template <int DK, int NW>
struct FwdStage {
  static constexpr int P = DK + 8, VP = NW * 16 + 8;
  bf16 k[C * P], q[C * P], v[C * VP], ap[4 * C * APITCH];
  float vec[SEQ_ROWS * 64];
};

// KEEP: also write what the backward pass needs; the results are the same, bit by bit.
template <int DK, int NW, bool KEEP>
__global__ void __launch_bounds__(NW * 32, 1)
forward_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Stage = FwdStage<DK, NW>;
  constexpr int P = Stage::P, VP = Stage::VP, THREADS = NW * 32, KT = DK / 16;
  Stage* st = reinterpret_cast<Stage*>(smem);
  const int splits = a.dv / (NW * 16);
  const int vb = blockIdx.x % splits, h = (blockIdx.x / splits) % a.Hv, n = blockIdx.x / (splits * a.Hv);
  const int hk = h / (a.Hv / a.Hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const int col0 = vb * NW * 16 + warp * 16;  // the warp's first column of dv
  const long long start = a.cu ? a.cu[n] : 0, end = a.cu ? a.cu[n + 1] : a.T, c0 = a.cu ? a.cbase[n] : 0;
  const int chunks = static_cast<int>((end - start + C - 1) / C);

  float s[2 * KT][4];  // S^T: rows = columns of dv, columns = dk
  const long long sbase = (static_cast<long long>(n) * a.Hv + h) * DK * a.dv + col0;
#pragma unroll
  for (int j = 0; j < 2 * KT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[j][e] = a.s_in ? a.s_in[sbase + static_cast<long long>(8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] : 0.f;

  auto fetch = [&](int c) {
    Stage& x = st[c & 1];
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const long long rec = (c0 + c) * a.Hv + h;
    load_rows<DK, THREADS>(x.k, P, static_cast<const bf16*>(a.k) + t0 * a.k_ts + hk * a.k_hs, a.k_ts, len);
    load_rows<DK, THREADS>(x.q, P, static_cast<const bf16*>(a.q) + t0 * a.q_ts + hk * a.q_hs, a.q_ts, len);
    load_rows<NW * 16, THREADS>(x.v, VP, static_cast<const bf16*>(a.v) + t0 * a.v_ts + h * a.v_hs + vb * NW * 16, a.v_ts, len);
    load_square<4, THREADS>(x.ap, static_cast<const bf16*>(a.ap) + rec * DELTA_AP);
    load_vec<THREADS>(x.vec, a.vec + rec * DELTA_VEC, SEQ_ROWS);
  };
  if (chunks > 0) fetch(0);
  cp_commit();
  for (int c = 0; c < chunks; ++c) {
    if (c + 1 < chunks) fetch(c + 1);
    cp_commit();
    cp_wait<1>();
    __syncthreads();
    Stage& x = st[c & 1];
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const bf16 *ahi = x.ap, *alo = x.ap + C * APITCH, *phi = x.ap + 2 * C * APITCH, *plo = x.ap + 3 * C * APITCH;
    uint4* sf = KEEP ? reinterpret_cast<uint4*>(a.states) + ((((c0 + c) * a.Hv + h) * (a.dv / 16) + (col0 >> 4)) * 2) * KT * 32 + lane : nullptr;

    bf16* stage = x.v + warp * 16;
    const long long out0 = (t0 * a.Hv + h) * a.dv + col0, ostride = static_cast<long long>(a.Hv) * a.dv;
    auto rest = [](float f) { return f - __bfloat162float(__float2bfloat16(f)); };

    // (K S)^T
    float u[8][4], y[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[j][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      uint32_t hi[4], lo[4], b[4][4];
      split_a(s[2 * kk], s[2 * kk + 1], hi, lo);
      if (KEEP) {
        sf[kk * 32] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        sf[(KT + kk) * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) b_from_nk(b[j], x.k, P, 16 * j, 16 * kk);
      mma2<4>(y, hi, lo, b);
    }
    // u <- beta (V - e^G K S)^T
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      uint32_t v[4];
      a_from_km(v, x.v, VP, 8 * j, warp * 16);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const int tok = 8 * (j + f) + t2;
        const float2 yk = *reinterpret_cast<const float2*>(x.vec + V_YK * 64 + tok);
        const float2 be = *reinterpret_cast<const float2*>(x.vec + V_BETA * 64 + tok);
        float(&z)[4] = y[j + f];
        z[0] *= yk.x;
        z[1] *= yk.y;
        z[2] *= yk.x;
        z[3] *= yk.y;
        u[j + f][0] = be.x * (lo_half(v[2 * f]) - z[0]);
        u[j + f][1] = be.y * (hi_half(v[2 * f]) - z[1]);
        u[j + f][2] = be.x * (lo_half(v[2 * f + 1]) - z[2]);
        u[j + f][3] = be.y * (hi_half(v[2 * f + 1]) - z[3]);
      }
    }
    // U^T = u + u (A - I)^T, from the last tokens to the first: column tile n needs the tiles up to n, so it may replace
    // its own. y becomes the memory read at each token, m = e^G K S - ((A - I) u) / beta, in 16 bits, and U is
    // beta (V - m), which the backward pass makes again from the m it reads: the products of dg must see the same U.
#pragma unroll
    for (int np = 3; np >= 0; --np) {
      float w[2][4];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[f][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk <= np; ++kk) {
        uint32_t hi[4], lo[4], b[4], c[4];
        split_a(u[2 * kk], u[2 * kk + 1], hi, lo);
        b_from_nk(b, ahi, APITCH, 16 * np, 16 * kk);
        b_from_nk(c, alo, APITCH, 16 * np, 16 * kk);
        mma(w[0], hi, b[0], b[1]);
        mma(w[1], hi, b[2], b[3]);
        mma(w[0], lo, b[0], b[1]);
        mma(w[1], lo, b[2], b[3]);
        mma(w[0], hi, c[0], c[1]);
        mma(w[1], hi, c[2], c[3]);
      }
      uint32_t v[4], mh[4], ml[4];
      a_from_km(v, x.v, VP, 16 * np, warp * 16);
      float m[2][4];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 be = *reinterpret_cast<const float2*>(x.vec + V_BETA * 64 + 16 * np + 8 * f + t2);
        m[f][0] = y[2 * np + f][0] - __fdividef(w[f][0], be.x);
        m[f][1] = y[2 * np + f][1] - __fdividef(w[f][1], be.y);
        m[f][2] = y[2 * np + f][2] - __fdividef(w[f][2], be.x);
        m[f][3] = y[2 * np + f][3] - __fdividef(w[f][3], be.y);
      }
      split_a(m[0], m[1], mh, ml);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 be = *reinterpret_cast<const float2*>(x.vec + V_BETA * 64 + 16 * np + 8 * f + t2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * f + e;
          memory_term(v[i], mh[i], ml[i], be, y[2 * np + f][2 * e], y[2 * np + f][2 * e + 1], u[2 * np + f][2 * e], u[2 * np + f][2 * e + 1]);
        }
      }
    }
    if (KEEP) {
      __syncwarp();
      store_tokens(stage, VP, static_cast<bf16*>(a.mem) + out0, ostride, len, [&](int j, int e) { return y[j][e]; });
      store_tokens(stage, VP, static_cast<bf16*>(a.mem_lo) + out0, ostride, len, [&](int j, int e) { return rest(y[j][e]); });
      store_tokens(stage, VP, static_cast<bf16*>(a.u) + out0, ostride, len, [&](int j, int e) { return u[j][e]; });
      store_tokens(stage, VP, static_cast<bf16*>(a.u_lo) + out0, ostride, len, [&](int j, int e) { return rest(u[j][e]); });
    }
    // what earlier tokens give to the output: e^G Q S + (P - diag P) U
    float(&o)[8][4] = y;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      uint32_t hi[4], lo[4], b[4][4];
      split_a(s[2 * kk], s[2 * kk + 1], hi, lo);
#pragma unroll
      for (int j = 0; j < 4; ++j) b_from_nk(b[j], x.q, P, 16 * j, 16 * kk);
      mma2<4>(o, hi, lo, b);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 oq = *reinterpret_cast<const float2*>(x.vec + V_OQ * 64 + 8 * j + t2);
      o[j][0] *= oq.x;
      o[j][1] *= oq.y;
      o[j][2] *= oq.x;
      o[j][3] *= oq.y;
    }
    // with U: its part of the output, and S^T <- e^{G_C} S^T + (e^{G_C - G} U)^T K
    const float ge = x.vec[V_END * 64];
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] *= ge;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4], b[4], c4[4];
      split_a(u[2 * kk], u[2 * kk + 1], hi, lo);
#pragma unroll
      for (int np = kk; np < 4; ++np) {  // all four parts: the backward pass multiplies with this P and this U too
        b_from_nk(b, phi, APITCH, 16 * np, 16 * kk);
        b_from_nk(c4, plo, APITCH, 16 * np, 16 * kk);
        mma(o[2 * np], hi, b[0], b[1]);
        mma(o[2 * np + 1], hi, b[2], b[3]);
        mma(o[2 * np], lo, b[0], b[1]);
        mma(o[2 * np + 1], lo, b[2], b[3]);
        mma(o[2 * np], hi, c4[0], c4[1]);
        mma(o[2 * np + 1], hi, c4[2], c4[3]);
        mma(o[2 * np], lo, c4[0], c4[1]);
        mma(o[2 * np + 1], lo, c4[2], c4[3]);
      }
      float w[2][4];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 su = *reinterpret_cast<const float2*>(x.vec + V_SU * 64 + 16 * kk + 8 * f + t2);
        w[f][0] = u[2 * kk + f][0] * su.x;
        w[f][1] = u[2 * kk + f][1] * su.y;
        w[f][2] = u[2 * kk + f][2] * su.x;
        w[f][3] = u[2 * kk + f][3] * su.y;
      }
      split_a(w[0], w[1], hi, lo);
#pragma unroll
      for (int j0 = 0; j0 < KT; j0 += 4) {
        uint32_t bs[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b_from_kn(bs[j], x.k, P, 16 * kk, 16 * (j0 + j));
        mma2<4>(s + 2 * j0, hi, lo, bs);
      }
    }
    if (KEEP) {  // eight neighbouring columns of a token per quarter of the warp: full 32-byte sectors
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tok = 8 * j + t2 + (e & 1);
          if (tok < len) a.past[out0 + tok * ostride + g + 8 * (e >> 1)] = o[j][e];
        }
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 pd = *reinterpret_cast<const float2*>(x.vec + V_PD * 64 + 8 * j + t2);
      o[j][0] += pd.x * u[j][0];
      o[j][1] += pd.y * u[j][1];
      o[j][2] += pd.x * u[j][2];
      o[j][3] += pd.y * u[j][3];
    }
    store_tokens(stage, VP, static_cast<bf16*>(a.o) + out0, ostride, len, [&](int j, int e) { return o[j][e]; });
    __syncthreads();  // the buffer is filled again in the next turn
  }
  cp_wait<0>();
  if (a.s_out) {
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        a.s_out[sbase + static_cast<long long>(8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] = s[j][e];
  }
}

// --------------------------------------------------------------------------------------------------------- backward

template <int DK, int NW>
struct BwdStage {
  static constexpr int P = DK + 8, VP = NW * 16 + 8;
  bf16 k[C * P], q[C * P], dO[C * VP], v[C * VP], m[C * VP], ml[C * VP], ap[4 * C * APITCH];
  float vec[SEQ_ROWS * 64];
};

template <int DK, int NW>
__global__ void __launch_bounds__(NW * 32, 1)
backward_kernel(const DeltaArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  using Stage = BwdStage<DK, NW>;
  constexpr int P = Stage::P, VP = Stage::VP, THREADS = NW * 32, KT = DK / 16;
  Stage* st = reinterpret_cast<Stage*>(smem);
  const int splits = a.dv / (NW * 16);
  const int vb = blockIdx.x % splits, h = (blockIdx.x / splits) % a.Hv, n = blockIdx.x / (splits * a.Hv);
  const int hk = h / (a.Hv / a.Hk);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const int col0 = vb * NW * 16 + warp * 16, VT = a.dv / 16, vt = col0 >> 4;
  const long long start = a.cu ? a.cu[n] : 0, end = a.cu ? a.cu[n + 1] : a.T, c0 = a.cu ? a.cbase[n] : 0;
  const int chunks = static_cast<int>((end - start + C - 1) / C);

  float s[2 * KT][4];  // dS^T
  const long long sbase = (static_cast<long long>(n) * a.Hv + h) * DK * a.dv + col0;
#pragma unroll
  for (int j = 0; j < 2 * KT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      s[j][e] = a.ds_out ? a.ds_out[sbase + static_cast<long long>(8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] : 0.f;

  auto fetch = [&](int c) {
    Stage& x = st[c & 1];
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const long long rec = (c0 + c) * a.Hv + h;
    const long long row = (t0 * a.Hv + h) * a.dv + vb * NW * 16, stride = static_cast<long long>(a.Hv) * a.dv;
    load_rows<DK, THREADS>(x.k, P, static_cast<const bf16*>(a.k) + t0 * a.k_ts + hk * a.k_hs, a.k_ts, len);
    load_rows<DK, THREADS>(x.q, P, static_cast<const bf16*>(a.q) + t0 * a.q_ts + hk * a.q_hs, a.q_ts, len);
    load_rows<NW * 16, THREADS>(x.dO, VP, static_cast<const bf16*>(a.dout) + row, stride, len);
    load_rows<NW * 16, THREADS>(x.v, VP, static_cast<const bf16*>(a.v) + t0 * a.v_ts + h * a.v_hs + vb * NW * 16, a.v_ts, len);
    load_rows<NW * 16, THREADS>(x.m, VP, static_cast<const bf16*>(a.mem) + row, stride, len);
    load_rows<NW * 16, THREADS>(x.ml, VP, static_cast<const bf16*>(a.mem_lo) + row, stride, len);
    load_square<4, THREADS>(x.ap, static_cast<const bf16*>(a.ap) + rec * DELTA_AP);
    load_vec<THREADS>(x.vec, a.vec + rec * DELTA_VEC, SEQ_ROWS);
  };
  if (chunks > 0) fetch(chunks - 1);
  cp_commit();
  for (int c = chunks - 1; c >= 0; --c) {
    if (c > 0) fetch(c - 1);
    cp_commit();
    cp_wait<1>();
    __syncthreads();
    Stage& x = st[c & 1];
    const long long t0 = start + static_cast<long long>(c) * C;
    const int len = end - t0 < C ? static_cast<int>(end - t0) : C;
    const long long rec = (c0 + c) * a.Hv + h;
    const bf16 *ahi = x.ap, *alo = x.ap + C * APITCH, *phi = x.ap + 2 * C * APITCH, *plo = x.ap + 3 * C * APITCH;
    uint4* df = reinterpret_cast<uint4*>(a.dstates) + (rec * VT + vt) * KT * 32 + lane;
    const uint4* nf = reinterpret_cast<const uint4*>(a.states) + ((rec * VT + vt) * 2) * KT * 32 + lane;

    // u = (e^{G_C - G} K dS1)^T; on the way <dS1, S0>
    float u[8][4], sdot = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) u[j][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      uint32_t hi[4], lo[4], b[4][4];
      split_a(s[2 * kk], s[2 * kk + 1], hi, lo);
      df[kk * 32] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      const uint4 qh = nf[kk * 32], ql = nf[(KT + kk) * 32];
      const uint32_t wh[4] = {qh.x, qh.y, qh.z, qh.w}, wl[4] = {ql.x, ql.y, ql.z, ql.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sdot += s[2 * kk + (e >> 1)][2 * (e & 1)] * (lo_half(wh[e]) + lo_half(wl[e]));
        sdot += s[2 * kk + (e >> 1)][2 * (e & 1) + 1] * (hi_half(wh[e]) + hi_half(wl[e]));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) b_from_nk(b[j], x.k, P, 16 * j, 16 * kk);
      mma2<4>(u, hi, lo, b);
    }
    const float ge = x.vec[V_END * 64];
    sdot *= ge;
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] *= ge;
    // Tiles j, j + 1 of the memory term m^T and of U^T = beta (V - m)^T
    auto load_mu = [&](int j, float(&mm)[2][4], float(&uu)[2][4]) {
      uint32_t fv[4], fm[4], fl[4];
      a_from_km(fv, x.v, VP, 8 * j, warp * 16);
      a_from_km(fm, x.m, VP, 8 * j, warp * 16);
      a_from_km(fl, x.ml, VP, 8 * j, warp * 16);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 be = *reinterpret_cast<const float2*>(x.vec + V_BETA * 64 + 8 * (j + f) + t2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * f + e;
          memory_term(fv[i], fm[i], fl[i], be, mm[f][2 * e], mm[f][2 * e + 1], uu[f][2 * e], uu[f][2 * e + 1]);
          uint32_t hi, lo;  // the two parts that the forward pass multiplied with P
          split2(uu[f][2 * e], uu[f][2 * e + 1], hi, lo);
          uu[f][2 * e] = lo_half(hi) + lo_half(lo);
          uu[f][2 * e + 1] = hi_half(hi) + hi_half(lo);
        }
      }
    };
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float mm[2][4], uu[2][4];
      load_mu(j, mm, uu);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 su = *reinterpret_cast<const float2*>(x.vec + V_SU * 64 + 8 * (j + f) + t2);
        u[j + f][0] *= su.x;
        u[j + f][1] *= su.y;
        u[j + f][2] *= su.x;
        u[j + f][3] *= su.y;
#pragma unroll
        for (int e = 0; e < 4; ++e) sdot += u[j + f][e] * uu[f][e];
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sdot += __shfl_xor_sync(0xffffffffu, sdot, o);
    if (lane == 0) a.sdots[rec * VT + vt] = sdot;
    // u += ((P - diag P)^T dO)^T, du = u + (diag P dO)^T = dU^T; and Q^T diag(e^G) dO into the state
    float du[8][4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t f[4], hi[4], lo[4], b[4];
      a_from_km(f, x.dO, VP, 16 * kk, warp * 16);
#pragma unroll
      for (int np = 0; np <= kk; ++np) {
        b_from_kn(b, phi, APITCH, 16 * kk, 16 * np);
        mma(u[2 * np], f, b[0], b[1]);
        mma(u[2 * np + 1], f, b[2], b[3]);
        b_from_kn(b, plo, APITCH, 16 * kk, 16 * np);
        mma(u[2 * np], f, b[0], b[1]);
        mma(u[2 * np + 1], f, b[2], b[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 pd = *reinterpret_cast<const float2*>(x.vec + V_PD * 64 + 16 * kk + 8 * (e >> 1) + t2);
        du[2 * kk + (e >> 1)][2 * (e & 1)] = pd.x * lo_half(f[e]);
        du[2 * kk + (e >> 1)][2 * (e & 1) + 1] = pd.y * hi_half(f[e]);
      }
      const float2 q0 = *reinterpret_cast<const float2*>(x.vec + V_OQ * 64 + 16 * kk + t2);
      const float2 q1 = *reinterpret_cast<const float2*>(x.vec + V_OQ * 64 + 16 * kk + 8 + t2);
      split2(lo_half(f[0]) * q0.x, hi_half(f[0]) * q0.y, hi[0], lo[0]);
      split2(lo_half(f[1]) * q0.x, hi_half(f[1]) * q0.y, hi[1], lo[1]);
      split2(lo_half(f[2]) * q1.x, hi_half(f[2]) * q1.y, hi[2], lo[2]);
      split2(lo_half(f[3]) * q1.x, hi_half(f[3]) * q1.y, hi[3], lo[3]);
#pragma unroll
      for (int j0 = 0; j0 < KT; j0 += 4) {
        uint32_t bs[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b_from_kn(bs[j], x.q, P, 16 * kk, 16 * (j0 + j));
        mma2<4>(s + 2 * j0, hi, lo, bs);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) du[j][e] += u[j][e];
    // u <- u + dU^T (A - I): X without what the token's own output asks for
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4], b[4];
      split_a(du[2 * kk], du[2 * kk + 1], hi, lo);
#pragma unroll
      for (int np = 0; np <= kk; ++np) {
        b_from_kn(b, ahi, APITCH, 16 * kk, 16 * np);
        mma(u[2 * np], hi, b[0], b[1]);
        mma(u[2 * np + 1], hi, b[2], b[3]);
        mma(u[2 * np], lo, b[0], b[1]);
        mma(u[2 * np + 1], lo, b[2], b[3]);
        b_from_kn(b, alo, APITCH, 16 * kk, 16 * np);
        mma(u[2 * np], hi, b[0], b[1]);
        mma(u[2 * np + 1], hi, b[2], b[3]);
      }
    }
    // X = u + (diag P dO)^T, and the row sums U . u, U . X and beta m . X over the warp's 16 columns
    float d[3][16];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float mm[2][4], uu[2][4];
      uint32_t fo[4];
      load_mu(j, mm, uu);
      a_from_km(fo, x.dO, VP, 8 * j, warp * 16);
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 pd = *reinterpret_cast<const float2*>(x.vec + V_PD * 64 + 8 * (j + f) + t2);
        const float2 be = *reinterpret_cast<const float2*>(x.vec + V_BETA * 64 + 8 * (j + f) + t2);
        float(&z)[4] = u[j + f];
        const int c0 = 2 * (j + f);
        d[0][c0] = uu[f][0] * z[0] + uu[f][2] * z[2];
        d[0][c0 + 1] = uu[f][1] * z[1] + uu[f][3] * z[3];
        z[0] += pd.x * lo_half(fo[2 * f]);
        z[1] += pd.y * hi_half(fo[2 * f]);
        z[2] += pd.x * lo_half(fo[2 * f + 1]);
        z[3] += pd.y * hi_half(fo[2 * f + 1]);
        d[1][c0] = uu[f][0] * z[0] + uu[f][2] * z[2];
        d[1][c0 + 1] = uu[f][1] * z[1] + uu[f][3] * z[3];
        z[0] *= be.x;  // dV = beta X
        z[1] *= be.y;
        z[2] *= be.x;
        z[3] *= be.y;
        d[2][c0] = mm[f][0] * z[0] + mm[f][2] * z[2];
        d[2][c0 + 1] = mm[f][1] * z[1] + mm[f][3] * z[3];
      }
    }
    float* rd = a.rowdots + (rec * VT + vt) * 192;
#pragma unroll
    for (int m = 0; m < 3; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float v = d[m][i];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) rd[m * 64 + 8 * (i >> 1) + t2 + (i & 1)] = v;
      }
    // dS0 -= K^T diag(e^G) dV
    __syncwarp();
    store_tokens(x.v + warp * 16, VP, static_cast<bf16*>(a.dv_) + (t0 * a.Hv + h) * a.dv + col0,
                 static_cast<long long>(a.Hv) * a.dv, len, [&](int j, int e) { return u[j][e]; });
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t hi[4], lo[4], b[4];
      float w[2][4];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float2 yk = *reinterpret_cast<const float2*>(x.vec + V_YK * 64 + 16 * kk + 8 * f + t2);
        w[f][0] = -u[2 * kk + f][0] * yk.x;
        w[f][1] = -u[2 * kk + f][1] * yk.y;
        w[f][2] = -u[2 * kk + f][2] * yk.x;
        w[f][3] = -u[2 * kk + f][3] * yk.y;
      }
      split_a(w[0], w[1], hi, lo);
#pragma unroll
      for (int j0 = 0; j0 < KT; j0 += 4) {
        uint32_t bs[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b_from_kn(bs[j], x.k, P, 16 * kk, 16 * (j0 + j));
        mma2<4>(s + 2 * j0, hi, lo, bs);
      }
    }
    __syncthreads();
  }
  cp_wait<0>();
  if (a.ds_in) {
#pragma unroll
    for (int j = 0; j < 2 * KT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        a.ds_in[sbase + static_cast<long long>(8 * j + t2 + (e & 1)) * a.dv + g + 8 * (e >> 1)] = s[j][e];
  }
}

// -------------------------------------------------------------------------------------------------------------- dqk

template <int DK, int DV>
struct DqkSmem {
  static constexpr int P = DK + 8, VP = DV + 8;
  bf16 q[C * P], k[C * P], dO[C * VP], dV[C * VP], u[C * VP], ul[C * VP], s0[DV * P], ds[DV * P];
  bf16 w1[C * APITCH], w1l[C * APITCH], w2[C * APITCH];
  float vec[8 * 64];
  float dots[2][2][C];
};

constexpr int DQK_THREADS = 256;

// State fragments of all dv / 16 column tiles -> [DV][DK] rows of pitch DK + 8.
template <int DK, int DV>
__device__ __forceinline__ void load_fragments(bf16* dst, const uint4* src, int tile_stride) {
  constexpr int KT = DK / 16, P = DK + 8;
  for (int i = threadIdx.x; i < DV / 16 * KT * 32; i += DQK_THREADS) {
    const int lane = i & 31, kk = (i >> 5) % KT, vt = (i >> 5) / KT, g = lane >> 2, t2 = (lane & 3) * 2;
    const uint4 f = src[static_cast<long long>(vt) * tile_stride + kk * 32 + lane];
    bf16* p = dst + (vt * 16 + g) * P + kk * 16 + t2;
    *reinterpret_cast<uint32_t*>(p) = f.x;
    *reinterpret_cast<uint32_t*>(p + 8 * P) = f.y;
    *reinterpret_cast<uint32_t*>(p + 8) = f.z;
    *reinterpret_cast<uint32_t*>(p + 8 * P + 8) = f.w;
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
  for (int hr = 0; hr < rep; ++hr) {
    const int h = hk * rep + hr;
    const long long rec = c * a.Hv + h;
    const long long row = (sp.start * a.Hv + h) * a.dv, stride = static_cast<long long>(a.Hv) * a.dv;
    __syncthreads();
    load_rows<DV, DQK_THREADS>(x.dO, VP, static_cast<const bf16*>(a.dout) + row, stride, sp.len);
    load_rows<DV, DQK_THREADS>(x.dV, VP, static_cast<const bf16*>(a.dv_) + row, stride, sp.len);
    load_rows<DV, DQK_THREADS>(x.u, VP, static_cast<const bf16*>(a.u) + row, stride, sp.len);
    load_rows<DV, DQK_THREADS>(x.ul, VP, static_cast<const bf16*>(a.u_lo) + row, stride, sp.len);
    load_vec<DQK_THREADS>(x.vec, a.vec + rec * DELTA_VEC, 8);
    cp_commit();
    load_fragments<DK, DV>(x.s0, reinterpret_cast<const uint4*>(a.states) + rec * (DV / 16) * 2 * KT * 32, 2 * KT * 32);
    load_fragments<DK, DV>(x.ds, reinterpret_cast<const uint4*>(a.dstates) + rec * (DV / 16) * KT * 32, KT * 32);
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
      uint32_t fo[4], fv[4], b[4], bl[4];
      a_from_mk(fo, x.dO, VP, wm * 16, kk * 16);
      a_from_mk(fv, x.dV, VP, wm * 16, kk * 16);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (wn * 2 + j > wm) continue;
        b_from_nk(b, x.u, VP, wn * 32 + j * 16, kk * 16);
        mma(p[2 * j], fo, b[0], b[1]);
        mma(p[2 * j + 1], fo, b[2], b[3]);
        mma(nn[2 * j], fv, b[0], b[1]);
        mma(nn[2 * j + 1], fv, b[2], b[3]);
        b_from_nk(bl, x.ul, VP, wn * 32 + j * 16, kk * 16);
        mma(p[2 * j], fo, bl[0], bl[1]);
        mma(p[2 * j + 1], fo, bl[2], bl[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (wn * 2 + (j >> 1) > wm) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = r0 + 8 * (e >> 1), jj = wn * 32 + j * 8 + t2 + (e & 1);
        float w1 = 0.f, w2 = 0.f;
        if (i >= jj) {
          const float d = x.vec[V_RK * 64 + jj] * __expf((x.vec[V_GHI * 64 + i] - x.vec[V_GHI * 64 + jj]) + (x.vec[V_GLO * 64 + i] - x.vec[V_GLO * 64 + jj]));
          w1 = x.vec[V_QS * 64 + i] * d * p[j][e];
          if (i > jj) w2 = -x.vec[V_RK * 64 + i] * d * nn[j][e];
        }
        const bf16 w1h = __float2bfloat16(w1);
        x.w1[i * APITCH + jj] = w1h;
        x.w1l[i * APITCH + jj] = __float2bfloat16(w1 - __bfloat162float(w1h));
        if (i >= jj) {  // N + N^T
          x.w2[i * APITCH + jj] = __float2bfloat16(w2);
          x.w2[jj * APITCH + i] = __float2bfloat16(w2);
        }
      }
    }
    // the products with the states: rows scaled afterwards
    float t[NT][4];
    auto clear = [&]() {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[j][e] = 0.f;
    };
    auto product = [&](const bf16* rows, const bf16* state) {
      clear();
#pragma unroll
      for (int kk = 0; kk < DV / 16; ++kk) {
        uint32_t f[4], b[4];
        a_from_mk(f, rows, VP, wm * 16, kk * 16);
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
    product(x.dO, x.s0);
    add(dq, x.vec[V_OQ * 64 + r0], x.vec[V_OQ * 64 + r0 + 8]);
    product(x.dV, x.s0);
    add(dk, -x.vec[V_YK * 64 + r0], -x.vec[V_YK * 64 + r0 + 8]);
    product(x.u, x.ds);
    add(dk, x.vec[V_SU * 64 + r0], x.vec[V_SU * 64 + r0 + 8]);
    __syncthreads();  // w1, w2
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint32_t f1[4], f1l[4], ft[4], ftl[4], f2[4], b[4];
      a_from_mk(f1, x.w1, APITCH, wm * 16, kk * 16);
      a_from_mk(f1l, x.w1l, APITCH, wm * 16, kk * 16);
      a_from_km(ft, x.w1, APITCH, kk * 16, wm * 16);
      a_from_km(ftl, x.w1l, APITCH, kk * 16, wm * 16);
      a_from_mk(f2, x.w2, APITCH, wm * 16, kk * 16);
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

// One block per (chunk, value head): o~ . do per token, then dbeta and the suffix sums of dg in 64 bits.
__global__ void __launch_bounds__(128)
gates_kernel(const DeltaArgs a) {
  __shared__ double od[C];
  const long long c = blockIdx.x / a.Hv;
  const int h = blockIdx.x % a.Hv;
  const Span sp = chunk_span(a, c);
  if (sp.len == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, VT = a.dv / 16;
  const long long rec = c * a.Hv + h;
  for (int i = warp; i < C; i += 4) {
    float s = 0.f;
    if (i < sp.len) {
      const long long row = ((sp.start + i) * a.Hv + h) * a.dv;
      for (int v = lane * 2; v < a.dv; v += 64) {
        const float2 p = *reinterpret_cast<const float2*>(a.past + row + v);
        const uint32_t d = *reinterpret_cast<const uint32_t*>(static_cast<const bf16*>(a.dout) + row + v);
        s += p.x * lo_half(d) + p.y * hi_half(d);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) od[i] = s;
  }
  __syncthreads();
  if (warp != 0) return;
  const float* rd = a.rowdots + rec * VT * 192;
  double carry = 0.0;
  for (int v = 0; v < VT; ++v) carry += a.sdots[rec * VT + v];
#pragma unroll
  for (int half = 1; half >= 0; --half) {
    const int i = half * 32 + lane;
    double later = 0.0, xu = 0.0, read = 0.0;
    for (int v = 0; v < VT; ++v) {
      later += rd[v * 192 + i];
      xu += rd[v * 192 + 64 + i];
      read += rd[v * 192 + 128 + i];
    }
    double s = od[i] - read - later;
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

template <typename K>
bool allow_smem(K kernel, size_t bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) == cudaSuccess;
}

template <int DK, int NW, bool KEEP>
int launch_forward(const DeltaArgs& a, cudaStream_t s) {
  const long long grid = static_cast<long long>(a.N) * a.Hv * (a.dv / (NW * 16));
  if (grid > INT32_MAX) return -2;
  const size_t bytes = 2 * sizeof(FwdStage<DK, NW>);
  if (!allow_smem(forward_kernel<DK, NW, KEEP>, bytes)) return -3;
  forward_kernel<DK, NW, KEEP><<<static_cast<unsigned>(grid), NW * 32, bytes, s>>>(a);
  return 0;
}

template <int DK, int NW>
int launch_backward(const DeltaArgs& a, cudaStream_t s) {
  const long long grid = static_cast<long long>(a.N) * a.Hv * (a.dv / (NW * 16));
  if (grid > INT32_MAX) return -2;
  const size_t bytes = 2 * sizeof(BwdStage<DK, NW>);
  if (!allow_smem(backward_kernel<DK, NW>, bytes)) return -3;
  backward_kernel<DK, NW><<<static_cast<unsigned>(grid), NW * 32, bytes, s>>>(a);
  return 0;
}

template <int DK, int DV>
int launch_dqk(const DeltaArgs& a, cudaStream_t s) {
  const size_t bytes = sizeof(DqkSmem<DK, DV>);
  if (!allow_smem(dqk_kernel<DK, DV>, bytes)) return -3;
  dqk_kernel<DK, DV><<<static_cast<unsigned>(a.NC * a.Hk), DQK_THREADS, bytes, s>>>(a);
  return 0;
}

template <int DK>
int forward_dk(const DeltaArgs& a, cudaStream_t s) {
  if (a.NC > 0) {
    const size_t bytes = (2 * C * (DK + 8)) * sizeof(bf16) + (2 * C * MP + 5 * C) * sizeof(float);
    if (!allow_smem(prepare_kernel<DK>, bytes)) return -3;
    prepare_kernel<DK><<<static_cast<unsigned>(a.NC * a.Hk), PREP_THREADS, bytes, s>>>(a);
  }
  const int rc = a.states ? launch_forward<DK, 4, true>(a, s) : launch_forward<DK, 4, false>(a, s);
  if (rc) return rc;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

template <int DK>
int backward_dk(const DeltaArgs& a, cudaStream_t s) {
  int rc = launch_backward<DK, 4>(a, s);
  if (rc) return rc;
  if (a.NC > 0) {
    rc = a.dv == 64 ? launch_dqk<DK, 64>(a, s) : launch_dqk<DK, 128>(a, s);
    if (rc) return rc;
    gates_kernel<<<static_cast<unsigned>(a.NC * a.Hv), 128, 0, s>>>(a);
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

void delta_zero_uncovered(const ZeroRows& z, const int* cu, int N, long long T, cudaStream_t s) {
  zero_rows_kernel<<<148, 256, 0, s>>>(z, cu, N, T);
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
