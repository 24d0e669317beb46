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
// Bound by memory. D / 8 lanes hold a head. A lane holds both elements of its rotated pairs (four of each half, 8 bytes
// at a time; eight neighbours behind the rotated span), so the rotation stays in the lane. A block takes a few tokens and
// lays (head, token) out so that a lane keeps one token, hence its cosines, for all its heads. The value (and gate) heads
// of the packed row are not touched forward; backward copies their gradients into the packed gradient, which is so
// written in one pass.
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
constexpr int AHEAD = 3, BAHEAD = 1;  // heads of a lane that are loaded before the first is worked on, forward and backward

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
    if (t >= a.T) {  // its lanes work on zeros
      cs[tk][f] = sn[tk][f] = 0.f;
      continue;
    }
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

// Where the lane's two groups of four elements lie in a head, and whether they rotate.
struct Place {
  int e0, e1, f0;  // f0: first of the four angles
  bool in;
};
__device__ __forceinline__ Place place(const QkNormRopeArgs& a, int hl) {
  Place p;
  const int half = a.rot_dim >> 1;
  if (a.interleaved) {
    p.e0 = 8 * hl;
    p.e1 = p.e0 + 4;
    p.in = p.e0 < a.rot_dim;
    p.f0 = 4 * hl;
  } else {
    p.in = 4 * hl < half;
    p.e0 = p.in ? 4 * hl : 8 * hl;  // behind the span: rot_dim + 8 (hl - half / 4)
    p.e1 = p.in ? half + 4 * hl : p.e0 + 4;
    p.f0 = 4 * hl;
  }
  if (!p.in) p.f0 = 0;
  return p;
}

struct Rotation {
  float c[4], s[4];
};
__device__ __forceinline__ Rotation rotation_of(const Place& p, const float* cs, const float* sn) {
  Rotation r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r.c[j] = p.in ? cs[p.f0 + j] : 1.f;
    r.s[j] = p.in ? sn[p.f0 + j] : 0.f;
  }
  return r;
}

// f[0..3] and f[4..7] are the lane's two groups; pairs are (j, j + 4), or (2j, 2j + 1) when interleaved.
__device__ __forceinline__ void rotate(float (&f)[8], const Rotation& r, int interleaved, float sign) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float s = sign * r.s[j];
    float& x = interleaved ? f[2 * j] : f[j];
    float& y = interleaved ? f[2 * j + 1] : f[j + 4];
    const float a = x * r.c[j] - y * s, b = y * r.c[j] + x * s;
    x = a;
    y = b;
  }
}

__device__ __forceinline__ void widen(const uint2& a, const uint2& b, float (&f)[8]) { unpack8(make_uint4(a.x, a.y, b.x, b.y), f); }

template <int LANES, bool IL>
__global__ void __launch_bounds__(THREADS)
qk_fwd_kernel(const QkNormRopeArgs a) {
  constexpr int D = LANES * 8, HEADS = THREADS / LANES;
  static_assert(HEADS % TOK == 0, "a lane keeps its token");
  __shared__ float cs[TOK][MAX_HALF], sn[TOK][MAX_HALF];
  const long long t0 = static_cast<long long>(blockIdx.x) * TOK;
  const int hl = threadIdx.x % LANES, slot = threadIdx.x / LANES, tk = slot % TOK;
  const Place pl = place(a, hl);
  const long long t = t0 + tk;
  const bool live = t < a.T;
  const int per = a.G * (a.R + 1);
  const bf16* row = static_cast<const bf16*>(a.x) + (live ? t : 0) * a.x_ts;
  uint2 lo[AHEAD], hi[AHEAD];
  auto fetch = [&](int hd0) {
#pragma unroll
    for (int w = 0; w < AHEAD; ++w) {
      const int hd = hd0 + w * (HEADS / TOK), grp = hd / (a.R + 1), r = hd - grp * (a.R + 1);
      const bf16* src = row + (grp * a.P + (r == a.R ? a.P - 2 : r)) * D;
      const bool ok = live && hd < per;
      lo[w] = ok ? *reinterpret_cast<const uint2*>(src + pl.e0) : make_uint2(0u, 0u);
      hi[w] = ok ? *reinterpret_cast<const uint2*>(src + pl.e1) : make_uint2(0u, 0u);
    }
  };
  fetch(slot / TOK);
  make_rotation(a, t0, cs, sn);
  float wq[8], wk[8];
  widen(*reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.qw) + pl.e0), *reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.qw) + pl.e1), wq);
  widen(*reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.kw) + pl.e0), *reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.kw) + pl.e1), wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] += a.w_offset;
    wk[j] += a.w_offset;
  }
  __syncthreads();
  const Rotation rot = rotation_of(pl, cs[tk], sn[tk]);
  // every lane of a warp makes the same number of turns: the sums over a head need them all
  const int turns = (per + AHEAD * (HEADS / TOK) - 1) / (AHEAD * (HEADS / TOK));
  for (int n = 0; n < turns; ++n) {
    const int hd0 = n * AHEAD * (HEADS / TOK) + slot / TOK;
    if (n > 0) fetch(hd0);
#pragma unroll
    for (int w = 0; w < AHEAD; ++w) {
      const int hd = hd0 + w * (HEADS / TOK), grp = hd / (a.R + 1), r = hd - grp * (a.R + 1);
      const bool is_k = r == a.R;
      float f[8];
      widen(lo[w], hi[w], f);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
      const float rstd = rsqrtf(head_sum<LANES>(ss) * (1.f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= rstd * (is_k ? wk[j] : wq[j]);
      rotate(f, rot, IL, 1.f);
      if (live && hd < per) {
        bf16* dst = is_k ? static_cast<bf16*>(a.k) + (t * a.G + grp) * D : static_cast<bf16*>(a.q) + (t * a.G * a.R + hd - grp) * D;
        const uint4 o = pack8(f);
        *reinterpret_cast<uint2*>(dst + pl.e0) = make_uint2(o.x, o.y);
        *reinterpret_cast<uint2*>(dst + pl.e1) = make_uint2(o.z, o.w);
      }
    }
  }
}

template <int LANES, bool IL>
__global__ void __launch_bounds__(THREADS, 3)
qk_bwd_kernel(const QkNormRopeArgs a) {
  constexpr int D = LANES * 8, HEADS = THREADS / LANES;
  __shared__ float cs[TOK][MAX_HALF], sn[TOK][MAX_HALF];
  __shared__ float red[HEADS][D];
  const int hl = threadIdx.x % LANES, slot = threadIdx.x / LANES, tk = slot % TOK;
  const Place pl = place(a, hl);
  float wq[8], wk[8], dwq[8], dwk[8];
  widen(*reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.qw) + pl.e0), *reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.qw) + pl.e1), wq);
  widen(*reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.kw) + pl.e0), *reinterpret_cast<const uint2*>(static_cast<const bf16*>(a.kw) + pl.e1), wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    wq[j] += a.w_offset;
    wk[j] += a.w_offset;
    dwq[j] = dwk[j] = 0.f;
  }
  const int per = a.G * a.P, turns = (per + BAHEAD * (HEADS / TOK) - 1) / (BAHEAD * (HEADS / TOK));
  for (long long t0 = static_cast<long long>(blockIdx.x) * TOK; t0 < a.T; t0 += static_cast<long long>(gridDim.x) * TOK) {
    const long long t = t0 + tk;
    const bool live = t < a.T;
    __syncthreads();
    make_rotation(a, t0, cs, sn);
    __syncthreads();
    const Rotation rot = rotation_of(pl, cs[tk], sn[tk]);
    const long long tl = live ? t : 0;
    const bf16* xrow = static_cast<const bf16*>(a.x) + tl * a.x_ts;
    const bf16* dq = static_cast<const bf16*>(a.dq) + tl * a.G * a.R * D;
    const bf16* dk = static_cast<const bf16*>(a.dk) + tl * a.G * D;
    const bf16* dv = static_cast<const bf16*>(a.dv) + tl * a.G * D;
    const bf16* dgate = static_cast<const bf16*>(a.dgate) + tl * a.G * a.R * D;
    bf16* dxrow = static_cast<bf16*>(a.dx) + tl * per * D;
    for (int n = 0; n < turns; ++n) {
      const int hd0 = n * BAHEAD * (HEADS / TOK) + slot / TOK;
      uint2 glo[BAHEAD], ghi[BAHEAD], xlo[BAHEAD], xhi[BAHEAD];
#pragma unroll
      for (int w = 0; w < BAHEAD; ++w) {
        const int hd = hd0 + w * (HEADS / TOK), grp = hd / a.P, p = hd - grp * a.P;
        const bf16* g = p < a.R ? dq + (grp * a.R + p) * D : p == a.P - 2 ? dk + grp * D : p == a.P - 1 ? dv + grp * D : dgate + (grp * a.R + p - a.R) * D;
        const bool ok = live && hd < per, turn = ok && (p < a.R || p == a.P - 2);
        const uint2 zero = make_uint2(0u, 0u);
        glo[w] = ok ? *reinterpret_cast<const uint2*>(g + pl.e0) : zero;
        ghi[w] = ok ? *reinterpret_cast<const uint2*>(g + pl.e1) : zero;
        xlo[w] = turn ? *reinterpret_cast<const uint2*>(xrow + hd * D + pl.e0) : zero;
        xhi[w] = turn ? *reinterpret_cast<const uint2*>(xrow + hd * D + pl.e1) : zero;
      }
#pragma unroll
      for (int w = 0; w < BAHEAD; ++w) {
        const int hd = hd0 + w * (HEADS / TOK), grp = hd / a.P, p = hd - grp * a.P;
        const bool is_k = p == a.P - 2, turn = p < a.R || is_k;
        float d[8], x[8];
        const uint2 zero = make_uint2(0u, 0u);
        widen(turn ? glo[w] : zero, turn ? ghi[w] : zero, d);
        widen(xlo[w], xhi[w], x);
        rotate(d, rot, IL, -1.f);
        // the two sums over the head: x . x and d w . x
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ss += x[j] * x[j];
          dot += d[j] * (is_k ? wk[j] : wq[j]) * x[j];
        }
        ss = head_sum<LANES>(ss);
        dot = head_sum<LANES>(dot);
        const float rstd = rsqrtf(ss * (1.f / D) + a.eps), m = dot * rstd * rstd * (1.f / D);
        const float rq = is_k ? 0.f : rstd, rk = is_k ? rstd : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // both are zero where nothing turns
          const float v = d[j] * x[j];
          dwq[j] += v * rq;
          dwk[j] += v * rk;
          d[j] = rstd * (d[j] * (is_k ? wk[j] : wq[j]) - x[j] * m);
        }
        if (live && hd < per) {
          const uint4 o = pack8(d);
          *reinterpret_cast<uint2*>(dxrow + hd * D + pl.e0) = turn ? make_uint2(o.x, o.y) : glo[w];
          *reinterpret_cast<uint2*>(dxrow + hd * D + pl.e1) = turn ? make_uint2(o.z, o.w) : ghi[w];
        }
      }
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      red[slot][pl.e0 + j] = which ? dwk[j] : dwq[j];
      red[slot][pl.e1 + j] = which ? dwk[j + 4] : dwq[j + 4];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += THREADS) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < HEADS; ++i) s += red[i][c];
      a.partial[(static_cast<long long>(blockIdx.x) * 2 + which) * D + c] = s;
    }
  }
}

// dw = sum over blocks of partial[b, ., c] in a fixed order: a block per 32 columns, 32 rows of threads.
__global__ void qk_dw_kernel(const float* __restrict__ partial, int blocks, int D, bf16* __restrict__ dqw, bf16* __restrict__ dkw) {
  __shared__ float red[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
#pragma unroll 8
  for (int b = threadIdx.y; b < blocks; b += 32) s += partial[static_cast<long long>(b) * 2 * D + c];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = red[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0) (col < D ? dqw[col] : dkw[col - D]) = __float2bfloat16(s);
}

template <int LANES>
void launch_fwd(const QkNormRopeArgs& a, unsigned grid, cudaStream_t s) {
  if (a.interleaved) qk_fwd_kernel<LANES, true><<<grid, THREADS, 0, s>>>(a);
  else qk_fwd_kernel<LANES, false><<<grid, THREADS, 0, s>>>(a);
}
template <int LANES>
void launch_bwd(const QkNormRopeArgs& a, int grid, cudaStream_t s) {
  if (a.interleaved) qk_bwd_kernel<LANES, true><<<grid, THREADS, 0, s>>>(a);
  else qk_bwd_kernel<LANES, false><<<grid, THREADS, 0, s>>>(a);
}

}  // namespace

int qk_norm_rope_bwd_grid(long long T) {
  const long long b = (T + TOK - 1) / TOK;
  return static_cast<int>(b < 148 * 3 ? b : 148 * 3);
}

int qk_norm_rope_fwd(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.rot_dim / 2 > MAX_HALF) return -1;
  if (a.T == 0) return 0;
  const long long grid = (a.T + TOK - 1) / TOK;
  if (grid > INT32_MAX) return -2;
  const unsigned gd = static_cast<unsigned>(grid);
  if (a.D == 64) launch_fwd<8>(a, gd, s);
  else if (a.D == 128) launch_fwd<16>(a, gd, s);
  else if (a.D == 256) launch_fwd<32>(a, gd, s);
  else return -1;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int qk_norm_rope_bwd(const QkNormRopeArgs& a, cudaStream_t s) {
  if (a.rot_dim / 2 > MAX_HALF || (a.D != 64 && a.D != 128 && a.D != 256)) return -1;
  const int grid = qk_norm_rope_bwd_grid(a.T);
  if (grid > 0) {
    if (a.D == 64) launch_bwd<8>(a, grid, s);
    else if (a.D == 128) launch_bwd<16>(a, grid, s);
    else launch_bwd<32>(a, grid, s);
  }
  qk_dw_kernel<<<2 * a.D / 32, dim3(32, 32), 0, s>>>(a.partial, grid, a.D, static_cast<bf16*>(a.dqw), static_cast<bf16*>(a.dkw));
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace lf
