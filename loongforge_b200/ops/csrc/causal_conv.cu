// Depthwise causal convolution over packed tokens, K = 2..4 taps, optional bias and SiLU, forward and backward, and
// its single-token form on a pool of windows.
//
//   p[t, c] = bias[c] + sum_i w[c, K - 1 - i] x[t - i, c]   (i <= position of t in its own sequence),  y = silu(p)
//   dp = dy silu'(p),  dx[s] = sum_i w[K - 1 - i] dp[s + i] (same sequence),  dw[K - 1 - i] = sum_t dp[t] x[t - i]
//
// Bound by memory: x is read and y written once. A thread owns a few neighbouring channels and walks down the tokens
// with the window in registers, so every row is read once plus a halo of K - 1 rows per block of tokens.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "linear_attn.h"

namespace lf {
namespace {

using bf16 = __nv_bfloat16;

template <int V> struct Vec;
template <> struct Vec<8> { using type = uint4; };
template <> struct Vec<4> { using type = uint2; };

template <int V>
__device__ __forceinline__ void unpack(const typename Vec<V>::type& q, float (&f)[V]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 t = __bfloat1622float2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <int V>
__device__ __forceinline__ typename Vec<V>::type pack(const float (&f)[V]) {
  typename Vec<V>::type q;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return q;
}

// Tokens of its own sequence in front of token t, capped at `most`; -1 when no sequence covers t.
__device__ __forceinline__ int earlier_tokens(const int* __restrict__ cu, int N, long long T, long long t, int most) {
  if (t >= T) return -1;
  if (cu == nullptr) return t < most ? static_cast<int>(t) : most;
  int lo = 0, hi = N;  // last n with cu[n] <= t
  if (t < cu[0] || t >= cu[N]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  const long long d = t - cu[lo];
  return d < most ? static_cast<int>(d) : most;
}

__device__ __forceinline__ float sigmoid(float p) { return __fdividef(1.f, 1.f + __expf(-p)); }

// Weights of V channels, taps last-to-first: wr[i] multiplies x[t - i].
template <int V, int K>
__device__ __forceinline__ void load_weights(const bf16* __restrict__ w, int c, float (&wr)[K][V]) {
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int i = 0; i < K; ++i) wr[i][j] = __bfloat162float(w[static_cast<long long>(c + j) * K + (K - 1 - i)]);
}

constexpr int FWD_THREADS = 128;
constexpr int FWD_ROWS = 16;

template <int K>
__global__ void __launch_bounds__(FWD_THREADS)
conv_fwd_kernel(const ConvArgs a, int cblocks) {
  constexpr int V = 8;
  __shared__ int front[FWD_ROWS];
  const long long t0 = static_cast<long long>(blockIdx.x / cblocks) * FWD_ROWS;
  const int c = ((blockIdx.x % cblocks) * FWD_THREADS + threadIdx.x) * V;
  if (threadIdx.x < FWD_ROWS) front[threadIdx.x] = earlier_tokens(a.cu, a.N, a.T, t0 + threadIdx.x, K - 1);
  __syncthreads();
  if (c >= a.C) return;
  const bf16* x = static_cast<const bf16*>(a.x) + c;
  bf16* y = static_cast<bf16*>(a.y) + c;
  float wr[K][V], bias[V], win[K][V];
  load_weights<V, K>(static_cast<const bf16*>(a.w), c, wr);
#pragma unroll
  for (int j = 0; j < V; ++j) bias[j] = a.bias ? __bfloat162float(static_cast<const bf16*>(a.bias)[c + j]) : 0.f;
  uint4 rows[FWD_ROWS];
  const int n = a.T - t0 < FWD_ROWS ? static_cast<int>(a.T - t0) : FWD_ROWS;
#pragma unroll
  for (int r = 0; r < FWD_ROWS; ++r)
    if (r < n) rows[r] = *reinterpret_cast<const uint4*>(x + (t0 + r) * a.x_ts);
#pragma unroll
  for (int i = 1; i < K; ++i) {  // win[i] = x[t - i]
    if (t0 - i >= 0) {
      unpack<V>(*reinterpret_cast<const uint4*>(x + (t0 - i) * a.x_ts), win[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) win[i][j] = 0.f;
    }
  }
#pragma unroll
  for (int r = 0; r < FWD_ROWS; ++r) {
    if (r >= n) break;
    const int f = front[r];
    unpack<V>(rows[r], win[0]);
    float p[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      p[j] = bias[j] + wr[0][j] * win[0][j];
#pragma unroll
      for (int i = 1; i < K; ++i)
        if (i <= f) p[j] += wr[i][j] * win[i][j];
      if (a.silu) p[j] *= sigmoid(p[j]);
      if (f < 0) p[j] = 0.f;
    }
    *reinterpret_cast<uint4*>(y + (t0 + r) * a.C) = pack<V>(p);
#pragma unroll
    for (int i = K - 1; i > 0; --i)
#pragma unroll
      for (int j = 0; j < V; ++j) win[i][j] = win[i - 1][j];
  }
}

// A block owns the rows [t0, t0 + span) of dx; it also visits the K - 1 rows behind them, whose dp reach back into the
// block, but adds to dw / db from its own rows only.
constexpr int BWD_THREADS = 128;
constexpr int BWD_V = 4;

template <int K>
__global__ void __launch_bounds__(BWD_THREADS)
conv_bwd_kernel(const ConvArgs a, int cblocks, int span) {
  constexpr int V = BWD_V, STEP = 8;
  using vec = typename Vec<V>::type;
  __shared__ int front[STEP];
  const int tb = blockIdx.x / cblocks;
  const long long t0 = static_cast<long long>(tb) * span;
  const int c = ((blockIdx.x % cblocks) * BWD_THREADS + threadIdx.x) * V;
  const bool act = c < a.C;
  const long long t1 = t0 + span < a.T ? t0 + span : a.T;  // first row behind the block's own
  const bf16* x = static_cast<const bf16*>(a.x) + c;
  const bf16* dy = static_cast<const bf16*>(a.dy) + c;
  bf16* dx = static_cast<bf16*>(a.dx) + c;
  float wr[K][V], bias[V], win[K][V], acc[K][V], dw[K][V], db[V];
  if (act) {
    load_weights<V, K>(static_cast<const bf16*>(a.w), c, wr);
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = a.bias ? __bfloat162float(static_cast<const bf16*>(a.bias)[c + j]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < K; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) win[i][j] = acc[i][j] = dw[i][j] = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) db[j] = 0.f;
  if (act) {
#pragma unroll
    for (int i = 1; i < K; ++i)
      if (t0 - i >= 0) unpack<V>(*reinterpret_cast<const vec*>(x + (t0 - i) * a.x_ts), win[i]);
  }
  for (long long tt = t0; tt < t1 + K - 1; tt += STEP) {
    __syncthreads();
    if (threadIdx.x < STEP) front[threadIdx.x] = earlier_tokens(a.cu, a.N, a.T, tt + threadIdx.x, K - 1);
    __syncthreads();
    if (!act) continue;
    vec xr[STEP], gr[STEP];
#pragma unroll
    for (int r = 0; r < STEP; ++r)
      if (tt + r < a.T && tt + r < t1 + K - 1) {
        xr[r] = *reinterpret_cast<const vec*>(x + (tt + r) * a.x_ts);
        gr[r] = *reinterpret_cast<const vec*>(dy + (tt + r) * a.C);
      }
#pragma unroll
    for (int r = 0; r < STEP; ++r) {
      const long long t = tt + r;
      if (t >= t1 + K - 1) break;
      const int f = front[r];
      const bool own = t < t1;
#pragma unroll
      for (int j = 0; j < V; ++j) acc[0][j] = 0.f;
      if (f >= 0) {  // a token of some sequence (so t < T)
        float g[V];
        unpack<V>(xr[r], win[0]);
        unpack<V>(gr[r], g);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float d = g[j];
          if (a.silu) {
            float p = bias[j] + wr[0][j] * win[0][j];
#pragma unroll
            for (int i = 1; i < K; ++i)
              if (i <= f) p += wr[i][j] * win[i][j];
            const float s = sigmoid(p);
            d *= s * (1.f + p * (1.f - s));
          }
#pragma unroll
          for (int i = 0; i < K; ++i)
            if (i <= f) {
              acc[i][j] += wr[i][j] * d;  // acc[i] belongs to row t - i
              if (own) dw[i][j] += d * win[i][j];
            }
          if (own) db[j] += d;
        }
      }
      const long long done = t - (K - 1);  // no later row reaches it
      if (done >= t0 && done < t1) *reinterpret_cast<vec*>(dx + done * a.C) = pack<V>(acc[K - 1]);
#pragma unroll
      for (int i = K - 1; i > 0; --i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          win[i][j] = win[i - 1][j];
          acc[i][j] = acc[i - 1][j];
        }
    }
  }
  if (!act) return;
  float* p = a.partial + static_cast<long long>(tb) * (K + 1) * a.C + c;
#pragma unroll
  for (int i = 0; i < K; ++i) *reinterpret_cast<float4*>(p + static_cast<long long>(i) * a.C) = make_float4(dw[i][0], dw[i][1], dw[i][2], dw[i][3]);
  *reinterpret_cast<float4*>(p + static_cast<long long>(K) * a.C) = make_float4(db[0], db[1], db[2], db[3]);
}

// dw[c, K - 1 - i] = sum over blocks of partial[b, i, c], in block order; db likewise from row K.
__global__ void conv_dw_kernel(const float* __restrict__ partial, int blocks, int C, int K, bf16* __restrict__ dw,
                               bf16* __restrict__ db) {
  const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long n = static_cast<long long>(K + 1) * C;
  if (idx >= n) return;
  float s = 0.f;
#pragma unroll 8
  for (int b = 0; b < blocks; ++b) s += partial[b * n + idx];
  const int i = static_cast<int>(idx / C), c = static_cast<int>(idx % C);
  if (i < K) dw[static_cast<long long>(c) * K + (K - 1 - i)] = __float2bfloat16(s);
  else if (db) db[c] = __float2bfloat16(s);
}

int bwd_span(long long T, int C) {
  // long enough that the fp32 partial sums stay a few per cent of the traffic, short enough for two blocks per SM
  const long long cblocks = (C + BWD_V * BWD_THREADS - 1) / (BWD_V * BWD_THREADS);
  int span = 128;
  while (span > 16 && (T + span - 1) / span * cblocks < 2 * 148) span >>= 1;
  return span;
}

constexpr int STEP_THREADS = 128;

template <int K>
__global__ void __launch_bounds__(STEP_THREADS)
conv_step_kernel(const ConvStepArgs a, int cblocks) {
  constexpr int V = 8;
  const int b = blockIdx.x / cblocks;
  const int c = ((blockIdx.x % cblocks) * STEP_THREADS + threadIdx.x) * V;
  long long slot = b;
  if (a.index) {
    slot = a.index[b];
    int again = 0;
    for (int i = threadIdx.x; i < b; i += STEP_THREADS) again |= a.index[i] == slot;
    again = __syncthreads_or(again);
    if (slot >= 0 && (again || slot >= a.slots)) {
      if (threadIdx.x == 0) *a.status = 7;
      slot = -1;
    }
  }
  if (c >= a.C) return;
  float p[V];
  if (slot < 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = 0.f;
  } else {
    uint4* st = reinterpret_cast<uint4*>(static_cast<bf16*>(a.state) + (slot * a.C + c) * (K - 1));
    uint4 raw[K - 1], wraw[K];
#pragma unroll
    for (int i = 0; i < K - 1; ++i) raw[i] = st[i];
    const uint4* wp = reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.w) + static_cast<long long>(c) * K);
#pragma unroll
    for (int i = 0; i < K; ++i) wraw[i] = wp[i];
    const uint4 xraw = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(a.x) + b * a.x_ts + c);
    const bf16* old = reinterpret_cast<const bf16*>(raw);
    const bf16* wt = reinterpret_cast<const bf16*>(wraw);
    const bf16* xn = reinterpret_cast<const bf16*>(&xraw);
    uint4 out[K - 1];
    bf16* nw = reinterpret_cast<bf16*>(out);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      p[j] = a.bias ? __bfloat162float(static_cast<const bf16*>(a.bias)[c + j]) : 0.f;
#pragma unroll
      for (int i = 0; i < K - 1; ++i) {
        p[j] += __bfloat162float(wt[j * K + i]) * __bfloat162float(old[j * (K - 1) + i]);
        nw[j * (K - 1) + i] = i + 1 < K - 1 ? old[j * (K - 1) + i + 1] : xn[j];
      }
      p[j] += __bfloat162float(wt[j * K + K - 1]) * __bfloat162float(xn[j]);
      if (a.silu) p[j] *= sigmoid(p[j]);
    }
#pragma unroll
    for (int i = 0; i < K - 1; ++i) st[i] = out[i];
  }
  *reinterpret_cast<uint4*>(static_cast<bf16*>(a.y) + static_cast<long long>(b) * a.C + c) = pack<V>(p);
}

}  // namespace

int conv_blocks(long long T, int C) {
  const int span = bwd_span(T, C);
  return static_cast<int>((T + span - 1) / span);
}

int conv_fwd(const ConvArgs& a, cudaStream_t s) {
  if (a.K < 2 || a.K > 4 || a.C % 8 != 0) return -1;
  if (a.T == 0) return 0;
  const int cblocks = (a.C + 8 * FWD_THREADS - 1) / (8 * FWD_THREADS);
  const long long grid = (a.T + FWD_ROWS - 1) / FWD_ROWS * cblocks;
  if (grid > INT32_MAX) return -2;
  const unsigned gd = static_cast<unsigned>(grid);
  if (a.K == 2) conv_fwd_kernel<2><<<gd, FWD_THREADS, 0, s>>>(a, cblocks);
  else if (a.K == 3) conv_fwd_kernel<3><<<gd, FWD_THREADS, 0, s>>>(a, cblocks);
  else conv_fwd_kernel<4><<<gd, FWD_THREADS, 0, s>>>(a, cblocks);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int conv_bwd(const ConvArgs& a, cudaStream_t s) {
  if (a.K < 2 || a.K > 4 || a.C % 8 != 0) return -1;
  const int span = bwd_span(a.T, a.C), blocks = conv_blocks(a.T, a.C);
  const int cblocks = (a.C + BWD_V * BWD_THREADS - 1) / (BWD_V * BWD_THREADS);
  const long long grid = static_cast<long long>(blocks) * cblocks;
  if (grid > INT32_MAX) return -2;
  if (grid > 0) {
    const unsigned gd = static_cast<unsigned>(grid);
    if (a.K == 2) conv_bwd_kernel<2><<<gd, BWD_THREADS, 0, s>>>(a, cblocks, span);
    else if (a.K == 3) conv_bwd_kernel<3><<<gd, BWD_THREADS, 0, s>>>(a, cblocks, span);
    else conv_bwd_kernel<4><<<gd, BWD_THREADS, 0, s>>>(a, cblocks, span);
  }
  const long long n = static_cast<long long>(a.K + 1) * a.C;
  conv_dw_kernel<<<static_cast<unsigned>((n + 127) / 128), 128, 0, s>>>(a.partial, blocks, a.C, a.K,
                                                                        static_cast<bf16*>(a.dw), static_cast<bf16*>(a.db));
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int conv_step(const ConvStepArgs& a, cudaStream_t s) {
  if (a.K < 2 || a.K > 4 || a.C % 8 != 0) return -1;
  if (a.B == 0) return 0;
  const int cblocks = (a.C + 8 * STEP_THREADS - 1) / (8 * STEP_THREADS);
  const long long grid = static_cast<long long>(a.B) * cblocks;
  if (grid > INT32_MAX) return -2;
  const unsigned gd = static_cast<unsigned>(grid);
  if (a.K == 2) conv_step_kernel<2><<<gd, STEP_THREADS, 0, s>>>(a, cblocks);
  else if (a.K == 3) conv_step_kernel<3><<<gd, STEP_THREADS, 0, s>>>(a, cblocks);
  else conv_step_kernel<4><<<gd, STEP_THREADS, 0, s>>>(a, cblocks);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace lf
