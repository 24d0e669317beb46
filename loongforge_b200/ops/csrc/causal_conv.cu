// Depthwise causal convolution over packed tokens, K = 2..4 taps, optional bias and SiLU, forward and backward, and
// its single-token form on a pool of windows.
//
//   p[t, c] = bias[c] + sum_i w[c, K - 1 - i] x[t - i, c]   (i <= position of t in its own sequence),  y = silu(p)
//   dp = dy silu'(p),  dx[s] = sum_i w[K - 1 - i] dp[s + i] (same sequence),  dw[K - 1 - i] = sum_t dp[t] x[t - i]
//
// Bound by memory: x is read and y written once. A thread owns a few neighbouring channels and walks down the tokens
// with the window in registers, so every row is read once plus a halo of K - 1 rows per block of tokens.
// 16384 x 8192: forward 98 us (5.5 TB/s), backward 180 us (4.5 TB/s, 60 % of the issue slots) + 7 for dw; 2047 x 6144: 15,
// 24 and 3 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "device_info.h"
#include "linear_attn.h"

namespace lf {
namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 q;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
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

// Two neighbouring channels in one 64-bit register pair: one instruction for both halves.
using f2 = unsigned long long;
__device__ __forceinline__ f2 make2(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 split(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 widen(uint32_t w) { return make2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t narrow(f2 v) {
  const float2 f = split(v);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 1 / (1 + 2^(-p log2 e)), without the steps that keep subnormal values: they vanish next to 1, and a quotient below
// 2^-126 is nothing beside bf16's steps.
__device__ __forceinline__ f2 sigmoid2(f2 p) {
  float2 f = split(mul2(p, make2(-1.4426950408889634f, -1.4426950408889634f)));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  f = split(add2(make2(f.x, f.y), make2(1.f, 1.f)));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.y));
  return make2(f.x, f.y);
}

constexpr int THREADS = 128;
// Channel pairs of a thread: the walk's addresses and tests are paid once for both (16384 x 8192 backward: 187 us with one,
// 175 with two).
constexpr int FV = 2, BV = 2;
// Rows that are loaded ahead of their use. 16384 x 8192: forward 96 us with 8 (104 with 4); backward holds two inputs, three
// windows and the sums of dw, so 4.
constexpr int FSTEP = 8, BSTEP = 4;
constexpr int MAX_SPAN = 128;

// The next STEP rows from p on into registers, of which there are `left`; p moves on.
template <typename T, int STEP>
__device__ __forceinline__ void load_rows(T (&r)[STEP], const bf16*& p, long long stride, int left) {
#pragma unroll
  for (int i = 0; i < STEP; ++i) {
    if (i < left) r[i] = *reinterpret_cast<const T*>(p);
    p += stride;
  }
}

template <int NV, int K>
__device__ __forceinline__ void load_pairs(const ConvArgs& a, int c, f2 (&wr)[K][NV], f2 (&bias)[NV]) {
  const bf16* w = static_cast<const bf16*>(a.w) + static_cast<long long>(c) * K;
  const bf16* b = static_cast<const bf16*>(a.bias) + c;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < K; ++i)  // wr[i] multiplies x[t - i]
      wr[i][j] = make2(__bfloat162float(w[2 * j * K + (K - 1 - i)]), __bfloat162float(w[(2 * j + 1) * K + (K - 1 - i)]));
    bias[j] = a.bias ? make2(__bfloat162float(b[2 * j]), __bfloat162float(b[2 * j + 1])) : 0ull;
  }
}

// A block owns `span` rows of THREADS * FV channel pairs. front[i]: see earlier_tokens; `plain` steps, those whose rows
// all have the whole window in their own sequence (nearly all of a long row), skip the tests for it.
template <int K>
__global__ void __launch_bounds__(THREADS)
conv_fwd_kernel(const ConvArgs a, int cblocks, int span) {
  static_assert(FV == 2, "two pairs a thread");
  constexpr int STEP = FSTEP;
  __shared__ int front[MAX_SPAN];
  const long long t0 = static_cast<long long>(blockIdx.x / cblocks) * span;
  const long long t1 = t0 + span < a.T ? t0 + span : a.T;
  const int c = ((blockIdx.x % cblocks) * THREADS + threadIdx.x) * 2 * FV;
  if (threadIdx.x < span) front[threadIdx.x] = earlier_tokens(a.cu, a.N, a.T, t0 + threadIdx.x, K - 1);
  __syncthreads();
  if (c >= a.C) return;
  const bf16* x = static_cast<const bf16*>(a.x) + c;
  bf16* y = static_cast<bf16*>(a.y) + c;
  f2 wr[K][FV], bias[FV], win[K][FV];
  uint2 rows0[STEP], rows1[STEP];
  const bf16* xt = x + t0 * a.x_ts;
  const int n = static_cast<int>(t1 - t0);
  load_rows(rows0, xt, a.x_ts, n);
  load_pairs<FV, K>(a, c, wr, bias);
#pragma unroll
  for (int i = 1; i < K; ++i) {  // win[i] = x[t - i]
    uint2 r = make_uint2(0u, 0u);
    if (t0 - i >= 0) r = *reinterpret_cast<const uint2*>(x + (t0 - i) * a.x_ts);
#pragma unroll
    for (int j = 0; j < FV; ++j) win[i][j] = widen(j ? r.y : r.x);
  }
  y += t0 * a.C;
  auto step = [&](int t, uint2 (&rows)[STEP], uint2 (&next)[STEP]) {
    load_rows(next, xt, a.x_ts, n - t - STEP);
    const int* f = front + t;
    bool plain = t + STEP <= n;
#pragma unroll
    for (int r = 0; r < STEP; ++r) plain = plain && f[r] == K - 1;
    auto row = [&](int r, int fr) {
      uint32_t out[FV];
#pragma unroll
      for (int j = 0; j < FV; ++j) {
        win[0][j] = widen(j ? rows[r].y : rows[r].x);
        f2 p = fma2(wr[0][j], win[0][j], bias[j]);
#pragma unroll
        for (int i = 1; i < K; ++i)
          if (i <= fr) p = fma2(wr[i][j], win[i][j], p);
        if (a.silu) p = mul2(p, sigmoid2(p));
        out[j] = fr < 0 ? 0u : narrow(p);
#pragma unroll
        for (int i = K - 1; i > 0; --i) win[i][j] = win[i - 1][j];
      }
      *reinterpret_cast<uint2*>(y) = make_uint2(out[0], out[1]);
      y += a.C;
    };
    if (plain) {
#pragma unroll
      for (int r = 0; r < STEP; ++r) row(r, K - 1);
    } else {
#pragma unroll
      for (int r = 0; r < STEP; ++r)
        if (t + r < n) row(r, f[r]);
    }
  };
  for (int t = 0; t < n; t += 2 * STEP) {  // two steps, so that the rows that came ahead need not move
    step(t, rows0, rows1);
    if (t + STEP < n) step(t + STEP, rows1, rows0);
  }
}

// The same walk for the gradients. A block owns the rows [t0, t1) of dx; it also visits the K - 1 rows behind them, whose
// dp reach back into the block, but adds to dw / db from its own rows only. acc[i] collects dx of row t - i.
template <int K>
__global__ void __launch_bounds__(THREADS)
conv_bwd_kernel(const ConvArgs a, int cblocks, int span) {
  static_assert(BV == 2, "two pairs a thread");
  constexpr int STEP = BSTEP;
  __shared__ int front[MAX_SPAN + STEP];
  const int tb = blockIdx.x / cblocks;
  const long long t0 = static_cast<long long>(tb) * span;
  const long long t1 = t0 + span < a.T ? t0 + span : a.T, t2 = t1 + K - 1 < a.T ? t1 + K - 1 : a.T;
  const int c = ((blockIdx.x % cblocks) * THREADS + threadIdx.x) * 2 * BV;
  for (int i = threadIdx.x; i < span + STEP; i += THREADS) front[i] = earlier_tokens(a.cu, a.N, a.T, t0 + i, K - 1);
  __syncthreads();
  if (c >= a.C) return;
  const bf16* x = static_cast<const bf16*>(a.x) + c;
  const bf16* dy = static_cast<const bf16*>(a.dy) + c;
  bf16* dx = static_cast<bf16*>(a.dx) + c;
  f2 wr[K][BV], bias[BV], win[K][BV], acc[K][BV], dw[K][BV], db[BV];
  uint2 xr[STEP], gr[STEP];
  const bf16 *xt = x + t0 * a.x_ts, *gt = dy + t0 * a.C;
  const int n = static_cast<int>(t1 - t0), n2 = static_cast<int>(t2 - t0);  // the block's rows, and with those behind
  load_rows(xr, xt, a.x_ts, n2);
  load_rows(gr, gt, a.C, n2);
  load_pairs<BV, K>(a, c, wr, bias);
#pragma unroll
  for (int i = 0; i < K; ++i) {
    uint2 r = make_uint2(0u, 0u);
    if (i > 0 && t0 - i >= 0) r = *reinterpret_cast<const uint2*>(x + (t0 - i) * a.x_ts);
#pragma unroll
    for (int j = 0; j < BV; ++j) {
      win[i][j] = widen(j ? r.y : r.x);
      acc[i][j] = dw[i][j] = db[j] = 0ull;
    }
  }
  dx += (t0 - (K - 1)) * a.C;
#pragma unroll 1
  for (int t = 0; t < n + K - 1; t += STEP) {
    uint2 nx[STEP], ng[STEP];
    load_rows(nx, xt, a.x_ts, n2 - t - STEP);
    load_rows(ng, gt, a.C, n2 - t - STEP);
    const int* f = front + t;
    bool plain = t + STEP <= n && t > 0;
#pragma unroll
    for (int r = 0; r < STEP; ++r) plain = plain && f[r] == K - 1;
    // `own`: the row is one of the block's; `out`: row t + r - (K - 1), which no later row reaches, is
    auto row = [&](int r, int fr, bool own, bool out) {
#pragma unroll
      for (int j = 0; j < BV; ++j) {
        acc[0][j] = 0ull;
        if (fr >= 0) {  // a token of some sequence
          win[0][j] = widen(j ? xr[r].y : xr[r].x);
          f2 d = widen(j ? gr[r].y : gr[r].x);
          if (a.silu) {
            f2 p = fma2(wr[0][j], win[0][j], bias[j]);
#pragma unroll
            for (int i = 1; i < K; ++i)
              if (i <= fr) p = fma2(wr[i][j], win[i][j], p);
            const f2 s = sigmoid2(p), ps = mul2(p, s);
            // silu' = s + p s (1 - s) = s + p s - (p s) s
            d = mul2(d, add2(s, fma2(mul2(ps, s), make2(-1.f, -1.f), ps)));
          }
#pragma unroll
          for (int i = 0; i < K; ++i)
            if (i <= fr) {
              acc[i][j] = fma2(wr[i][j], d, acc[i][j]);
              if (own) dw[i][j] = fma2(d, win[i][j], dw[i][j]);
            }
          if (own) db[j] = add2(db[j], d);
        }
      }
      if (out) *reinterpret_cast<uint2*>(dx) = make_uint2(narrow(acc[K - 1][0]), narrow(acc[K - 1][1]));
      dx += a.C;
#pragma unroll
      for (int i = K - 1; i > 0; --i)
#pragma unroll
        for (int j = 0; j < BV; ++j) {
          win[i][j] = win[i - 1][j];
          acc[i][j] = acc[i - 1][j];
        }
    };
    if (plain) {
#pragma unroll
      for (int r = 0; r < STEP; ++r) row(r, K - 1, true, true);
    } else {
#pragma unroll
      for (int r = 0; r < STEP; ++r)
        if (t + r < n + K - 1) row(r, f[r], t + r < n, t + r >= K - 1);
    }
#pragma unroll
    for (int r = 0; r < STEP; ++r) {
      xr[r] = nx[r];
      gr[r] = ng[r];
    }
  }
  float* p = a.partial + static_cast<long long>(tb) * (K + 1) * a.C + c;
#pragma unroll
  for (int i = 0; i <= K; ++i) {
    const float2 u = split(i < K ? dw[i][0] : db[0]), v = split(i < K ? dw[i][1] : db[1]);
    *reinterpret_cast<float4*>(p + static_cast<long long>(i) * a.C) = make_float4(u.x, u.y, v.x, v.y);
  }
}

// dw[c, K - 1 - i] = sum over blocks of partial[b, i, c], in a fixed order; db likewise from row K. Eight threads share a
// column, which is a matter of latency: 7 us instead of 18 for 128 blocks of 8192 channels.
constexpr int DW_COLS = 32, DW_ROWS = 8;

__global__ void __launch_bounds__(DW_COLS * DW_ROWS)
conv_dw_kernel(const float* __restrict__ partial, int blocks, int C, int K, bf16* __restrict__ dw, bf16* __restrict__ db) {
  __shared__ float red[DW_ROWS][DW_COLS];
  const long long idx = static_cast<long long>(blockIdx.x) * DW_COLS + threadIdx.x;
  const long long n = static_cast<long long>(K + 1) * C;
  float s = 0.f;
  if (idx < n) {
#pragma unroll 8
    for (int b = threadIdx.y; b < blocks; b += DW_ROWS) s += partial[b * n + idx];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y != 0 || idx >= n) return;
#pragma unroll
  for (int r = 1; r < DW_ROWS; ++r) s += red[r][threadIdx.x];
  const int i = static_cast<int>(idx / C), c = static_cast<int>(idx % C);
  if (i < K) dw[static_cast<long long>(c) * K + (K - 1 - i)] = __float2bfloat16(s);
  else if (db) db[c] = __float2bfloat16(s);
}

// Rows of a block: long, so that halo rows and the fp32 partial sums of dw stay a few per cent of the traffic, but short
// enough that there are two blocks per SM.
int row_span(long long T, int C, int v) {
  const long long cblocks = (C + 2 * v * THREADS - 1) / (2 * v * THREADS);
  const int blocks = 2 * sm_count();
  int span = MAX_SPAN;
  while (span > 16 && (T + span - 1) / span * cblocks < blocks) span >>= 1;
  return span;
}

constexpr int STEP_THREADS = 128;

template <int K>
__global__ void __launch_bounds__(STEP_THREADS)
conv_step_kernel(const ConvStepArgs a, int cblocks) {
  constexpr int V = 8;  // channels of a thread: 16-byte pieces of x, state and weights
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
  *reinterpret_cast<uint4*>(static_cast<bf16*>(a.y) + static_cast<long long>(b) * a.C + c) = pack8(p);
}

}  // namespace

int conv_blocks(long long T, int C) {
  const int span = row_span(T, C, BV);
  return static_cast<int>((T + span - 1) / span);
}

int conv_fwd(const ConvArgs& a, cudaStream_t s) {
  if (a.K < 2 || a.K > 4 || a.C % 8 != 0) return -1;
  const int cblocks = (a.C + 2 * FV * THREADS - 1) / (2 * FV * THREADS), span = row_span(a.T, a.C, FV);
  const long long grid = (a.T + span - 1) / span * cblocks;
  if (grid > INT32_MAX) return -2;
  if (grid == 0) return 0;
  const unsigned gd = static_cast<unsigned>(grid);
  if (a.K == 2) conv_fwd_kernel<2><<<gd, THREADS, 0, s>>>(a, cblocks, span);
  else if (a.K == 3) conv_fwd_kernel<3><<<gd, THREADS, 0, s>>>(a, cblocks, span);
  else conv_fwd_kernel<4><<<gd, THREADS, 0, s>>>(a, cblocks, span);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int conv_bwd(const ConvArgs& a, cudaStream_t s) {
  if (a.K < 2 || a.K > 4 || a.C % 8 != 0) return -1;
  const int cblocks = (a.C + 2 * BV * THREADS - 1) / (2 * BV * THREADS), span = row_span(a.T, a.C, BV), blocks = conv_blocks(a.T, a.C);
  const long long grid = static_cast<long long>(blocks) * cblocks;
  if (grid > INT32_MAX) return -2;
  if (grid > 0) {
    const unsigned gd = static_cast<unsigned>(grid);
    if (a.K == 2) conv_bwd_kernel<2><<<gd, THREADS, 0, s>>>(a, cblocks, span);
    else if (a.K == 3) conv_bwd_kernel<3><<<gd, THREADS, 0, s>>>(a, cblocks, span);
    else conv_bwd_kernel<4><<<gd, THREADS, 0, s>>>(a, cblocks, span);
  }
  const long long n = static_cast<long long>(a.K + 1) * a.C;
  conv_dw_kernel<<<static_cast<unsigned>((n + DW_COLS - 1) / DW_COLS), dim3(DW_COLS, DW_ROWS), 0, s>>>(
      a.partial, blocks, a.C, a.K, static_cast<bf16*>(a.dw), static_cast<bf16*>(a.db));
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
