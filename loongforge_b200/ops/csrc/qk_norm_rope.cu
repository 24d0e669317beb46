// RMS norm of every query and key head with the position rotation in the same pass, straight out of the packed
// projection [T, groups, heads of a group, D], forward and backward.
//
//   n = x rstd (w + off),  rstd = (mean(x^2) + eps)^-1/2;  y = R(angle) n  on the first rot_dim elements, n behind them
//   backward: d = R(-angle) dy;  dw = sum d x rstd;  dx = rstd (d (w + off)) - x rstd^3 mean(d (w + off) x)
//
// Angles come from a table row per token, or as position[axis[i], t] * inv_freq[i] with one, two or three position axes
// (time, height, width). They are reduced to turns in 64 bits before sine and cosine: positions far into a long
// context keep their fraction.
//
// Bound by memory. D / 8 lanes hold a head, 16 bytes each; the rotation's partner elements are a shuffle away. The
// cosines of a few tokens are made once per block and shared by all their heads. The value (and gate) heads of the
// packed row are not touched forward; backward copies their gradients into the packed gradient, which is so written in
// one pass.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "elementwise.h"

namespace lf {
namespace {

using bf16 = __nv_bfloat16;
constexpr int THREADS = 256;
constexpr int TOK = 4;       // tokens of a block's turn
constexpr int MAX_HALF = 128;

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 q;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return q;
}

template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cos / sin of TOK tokens from t0 into shared memory.
__device__ __forceinline__ void make_rotation(const QkNormRopeArgs& a, long long t0, float (*cs)[MAX_HALF], float (*sn)[MAX_HALF]) {
  const int half = a.rot_dim >> 1;
  for (int i = threadIdx.x; i < TOK * half; i += THREADS) {
    const int tk = i / half, f = i - tk * half;
    const long long t = t0 + tk;
    if (t >= a.T) continue;
    double ang = 0.0;
    if (a.freqs) {
      const long long row = a.pos ? a.pos[t] : t;
      if (row >= 0 && row < a.freq_rows) ang = a.freqs[row * half + f];
      else *a.status = 7;
    } else {
      const int ax = a.axis ? a.axis[f] : 0;
      if (ax >= 0 && ax < a.axes) ang = static_cast<double>(a.pos[static_cast<long long>(ax) * a.T + t]) * static_cast<double>(a.inv_freq[f]);
      else *a.status = 7;
    }
    const double turns = ang * 0.15915494309189533577;
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    cs[tk][f] = c * a.mscale;
    sn[tk][f] = s * a.mscale;
  }
}

// Rotates the thread's eight elements [8 * hl, 8 * hl + 8) of a head by sign * angle; all lanes of the warp call it.
template <int LANES>
__device__ __forceinline__ void rotate(float (&f)[8], int hl, const float* cs, const float* sn, int rot_dim, int interleaved, float sign) {
  const int e0 = hl * 8;
  if (interleaved) {
    if (e0 < rot_dim) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float c = cs[e0 / 2 + j], s = sign * sn[e0 / 2 + j], x = f[2 * j], y = f[2 * j + 1];
        f[2 * j] = x * c - y * s;
        f[2 * j + 1] = y * c + x * s;
      }
    }
    return;
  }
  const int half = rot_dim >> 1, step = half >> 3;
  const bool in = e0 < rot_dim, upper = e0 >= half;
  const int partner = in ? (upper ? hl - step : hl + step) : hl;
  const int src = (threadIdx.x & 31 & ~(LANES - 1)) + partner;
  const int i0 = in ? (upper ? e0 - half : e0) : 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float other = __shfl_sync(0xffffffffu, f[j], src);
    if (in) {
      const float c = cs[i0 + j], s = sign * sn[i0 + j];
      f[j] = upper ? f[j] * c + other * s : f[j] * c - other * s;
    }
  }
}

template <int LANES>
__global__ void __launch_bounds__(THREADS)
qk_fwd_kernel(const QkNormRopeArgs a) {
  constexpr int D = LANES * 8, HEADS = THREADS / LANES;
  __shared__ float cs[TOK][MAX_HALF], sn[TOK][MAX_HALF];
  const long long t0 = static_cast<long long>(blockIdx.x) * TOK;
  make_rotation(a, t0, cs, sn);
  const int hl = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  float wq[8], wk[8];
  unpack8(reinterpret_cast<const uint4*>(a.qw)[hl], wq);
  unpack8(reinterpret_cast<const uint4*>(a.kw)[hl], wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] += a.w_offset;
    wk[j] += a.w_offset;
  }
  __syncthreads();
  const int per = a.G * (a.R + 1), n = static_cast<int>(a.T - t0 < TOK ? a.T - t0 : TOK) * per;
  // the loop runs the same number of turns in every lane of a warp: shuffles need them all
  for (int base = 0; base < n; base += HEADS) {
    const int idx = base + slot;
    const bool act = idx < n;
    const int tk = act ? idx / per : 0, hd = act ? idx - tk * per : 0;
    const int grp = hd / (a.R + 1), r = hd - grp * (a.R + 1);
    const bool is_k = r == a.R;
    const long long t = t0 + tk;
    const bf16* src = static_cast<const bf16*>(a.x) + t * a.x_ts + (static_cast<long long>(grp) * a.P + (is_k ? a.P - 2 : r)) * D;
    float f[8];
    unpack8(act ? reinterpret_cast<const uint4*>(src)[hl] : make_uint4(0u, 0u, 0u, 0u), f);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
    const float rstd = rsqrtf(head_sum<LANES>(ss) / static_cast<float>(D) + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= rstd * (is_k ? wk[j] : wq[j]);
    rotate<LANES>(f, hl, cs[tk], sn[tk], a.rot_dim, a.interleaved, 1.f);
    if (act) {
      bf16* dst = is_k ? static_cast<bf16*>(a.k) + (t * a.G + grp) * D : static_cast<bf16*>(a.q) + (t * a.G * a.R + grp * a.R + r) * D;
      reinterpret_cast<uint4*>(dst)[hl] = pack8(f);
    }
  }
}

template <int LANES>
__global__ void __launch_bounds__(THREADS)
qk_bwd_kernel(const QkNormRopeArgs a) {
  constexpr int D = LANES * 8, HEADS = THREADS / LANES;
  __shared__ float cs[TOK][MAX_HALF], sn[TOK][MAX_HALF];
  __shared__ float red[HEADS][D];
  const int hl = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  float wq[8], wk[8], dwq[8], dwk[8];
  unpack8(reinterpret_cast<const uint4*>(a.qw)[hl], wq);
  unpack8(reinterpret_cast<const uint4*>(a.kw)[hl], wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] += a.w_offset;
    wk[j] += a.w_offset;
    dwq[j] = dwk[j] = 0.f;
  }
  const int per = a.G * a.P;
  for (long long t0 = static_cast<long long>(blockIdx.x) * TOK; t0 < a.T; t0 += static_cast<long long>(gridDim.x) * TOK) {
    __syncthreads();
    make_rotation(a, t0, cs, sn);
    __syncthreads();
    const int n = static_cast<int>(a.T - t0 < TOK ? a.T - t0 : TOK) * per;
    for (int base = 0; base < n; base += HEADS) {
      const int idx = base + slot;
      const bool act = idx < n;
      const int tk = act ? idx / per : 0, hd = act ? idx - tk * per : 0;
      const int grp = hd / a.P, p = hd - grp * a.P;
      const bool is_q = p < a.R, is_k = p == a.P - 2, is_v = p == a.P - 1;
      const long long t = t0 + tk;
      const bf16* g;
      if (is_q) g = static_cast<const bf16*>(a.dq) + (t * a.G * a.R + grp * a.R + p) * D;
      else if (is_k) g = static_cast<const bf16*>(a.dk) + (t * a.G + grp) * D;
      else if (is_v) g = static_cast<const bf16*>(a.dv) + (t * a.G + grp) * D;
      else g = static_cast<const bf16*>(a.dgate) + (t * a.G * a.R + grp * a.R + p - a.R) * D;
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      const bool turn = act && (is_q || is_k);
      const uint4 graw = act ? reinterpret_cast<const uint4*>(g)[hl] : zero;
      const uint4 xraw = turn ? reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.x) + t * a.x_ts + static_cast<long long>(hd) * D)[hl] : zero;
      uint4* dst = reinterpret_cast<uint4*>(static_cast<bf16*>(a.dx) + (t * per + hd) * D) + hl;
      float d[8], x[8];
      unpack8(graw, d);
      unpack8(xraw, x);
      rotate<LANES>(d, hl, cs[tk], sn[tk], a.rot_dim, a.interleaved, -1.f);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
      const float rstd = rsqrtf(head_sum<LANES>(ss) / static_cast<float>(D) + a.eps);
      float dot = 0.f;
      if (turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = d[j] * x[j] * rstd;
          if (is_k) dwk[j] += w; else dwq[j] += w;
          d[j] *= is_k ? wk[j] : wq[j];
          dot += d[j] * x[j];
        }
      }
      dot = head_sum<LANES>(dot) * rstd * rstd / static_cast<float>(D);
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = rstd * (d[j] - x[j] * dot);
      if (act) *dst = turn ? pack8(d) : graw;
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) red[slot][hl * 8 + j] = which ? dwk[j] : dwq[j];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += THREADS) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < HEADS; ++i) s += red[i][c];
      a.partial[(static_cast<long long>(blockIdx.x) * 2 + which) * D + c] = s;
    }
  }
}

// dw = sum over blocks of partial[b, ., c] in a fixed order: a block per 32 columns, 8 rows of threads.
__global__ void qk_dw_kernel(const float* __restrict__ partial, int blocks, int D, bf16* __restrict__ dqw, bf16* __restrict__ dkw) {
  __shared__ float red[8][32];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  for (int b = threadIdx.y; b < blocks; b += 8) s += partial[static_cast<long long>(b) * 2 * D + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[i][threadIdx.x];
    (c < D ? dqw[c] : dkw[c - D]) = __float2bfloat16(s);
  }
}

}  // namespace

int qk_norm_rope_bwd_grid(long long T) {
  const long long b = (T + TOK - 1) / TOK;
  return static_cast<int>(b < 148 * 4 ? b : 148 * 4);
}

int qk_norm_rope_fwd(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.rot_dim / 2 > MAX_HALF) return -1;
  if (a.T == 0) return 0;
  const long long grid = (a.T + TOK - 1) / TOK;
  if (grid > INT32_MAX) return -2;
  const unsigned gd = static_cast<unsigned>(grid);
  if (a.D == 64) qk_fwd_kernel<8><<<gd, THREADS, 0, s>>>(a);
  else if (a.D == 128) qk_fwd_kernel<16><<<gd, THREADS, 0, s>>>(a);
  else if (a.D == 256) qk_fwd_kernel<32><<<gd, THREADS, 0, s>>>(a);
  else return -1;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int qk_norm_rope_bwd(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.rot_dim / 2 > MAX_HALF || (a.D != 64 && a.D != 128 && a.D != 256)) return -1;
  const int grid = qk_norm_rope_bwd_grid(a.T);
  if (grid > 0) {
    if (a.D == 64) qk_bwd_kernel<8><<<grid, THREADS, 0, s>>>(a);
    else if (a.D == 128) qk_bwd_kernel<16><<<grid, THREADS, 0, s>>>(a);
    else qk_bwd_kernel<32><<<grid, THREADS, 0, s>>>(a);
  }
  qk_dw_kernel<<<2 * a.D / 32, dim3(32, 8), 0, s>>>(a.partial, grid, a.D, static_cast<bf16*>(a.dqw), static_cast<bf16*>(a.dkw));
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace lf
