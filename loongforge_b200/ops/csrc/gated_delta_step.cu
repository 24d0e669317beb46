// Single-token form of the gated delta rule on a pool of fp32 states [slots, Hv, dk, dv], updated in place:
//
//   S <- a S,  u = beta (v - S^T k),  S <- S + k u^T,  o = S^T q       (a = e^g; q scaled, q and k normalised)
//
// Both products with the old state are taken in one pass, o = a S_old^T q + (k.q) u, so the state is read once, held in
// registers across one reduction over dk, and written once. Bound by memory: 8 dk dv bytes per row and head.
// A block takes COLS of the dv columns of one (row, head): the columns are independent, so few rows are cut into more
// blocks until the SMs are full.
// 192 rows of 48 heads of 128 x 128: 210 us, 5.8 TB/s; one row of 32 heads: 4.5 us, which is launch and one trip to memory.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "device_info.h"
#include "linear_attn.h"

namespace lf {
namespace {

using bf16 = __nv_bfloat16;
constexpr int THREADS = 256;

template <int DK, int COLS>
__global__ void __launch_bounds__(THREADS)
delta_step_kernel(const DeltaStepArgs a) {
  constexpr int CT = COLS / 4;            // threads across the columns, a float4 each
  constexpr int GROUPS = THREADS / CT;    // row groups
  constexpr int ROWS = DK / GROUPS;       // rows of one thread: r * GROUPS + group
  constexpr int WARPS = THREADS / 32;
  __shared__ float qs[DK], ks[DK], part[2][WARPS][COLS], norms[3][WARPS];
  const int splits = a.dv / COLS;
  const int vb = blockIdx.x % splits, h = (blockIdx.x / splits) % a.Hv, b = blockIdx.x / (splits * a.Hv);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long slot = b;
  if (a.index) {
    // a negative slot is a padding row; a slot out of range, or one that an earlier row has, is reported and skipped
    slot = a.index[b];
    int again = 0;
    for (int i = tid; i < b; i += THREADS) again |= a.index[i] == slot;
    again = __syncthreads_or(again);
    if (slot >= 0 && (again || slot >= a.slots)) {
      if (tid == 0) *a.status = 7;
      slot = -1;
    }
  }
  bf16* o = static_cast<bf16*>(a.o) + (static_cast<long long>(b) * a.Hv + h) * a.dv + vb * COLS;
  if (slot < 0) {
    if (tid < COLS) o[tid] = __float2bfloat16(0.f);
    return;
  }
  const int col = (tid % CT) * 4, grp = tid / CT;
  float4* S = reinterpret_cast<float4*>(a.state + ((slot * a.Hv + h) * DK) * a.dv + vb * COLS + col);
  const long long ld = a.dv / 4;
  float4 s[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) s[r] = S[(r * GROUPS + grp) * ld];
  const int hk = h / (a.Hv / a.Hk);
  float qv = 0.f, kv = 0.f;
  if (tid < DK) {
    qv = __bfloat162float(static_cast<const bf16*>(a.q)[b * a.q_ts + hk * a.q_hs + tid]);
    kv = __bfloat162float(static_cast<const bf16*>(a.k)[b * a.k_ts + hk * a.k_hs + tid]);
  }
  float n0 = qv * qv, n1 = kv * kv, n2 = qv * kv;
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) {
    n0 += __shfl_xor_sync(0xffffffffu, n0, i);
    n1 += __shfl_xor_sync(0xffffffffu, n1, i);
    n2 += __shfl_xor_sync(0xffffffffu, n2, i);
  }
  if (lane == 0) {
    norms[0][warp] = n0;
    norms[1][warp] = n1;
    norms[2][warp] = n2;
  }
  if (tid < DK) {
    qs[tid] = qv;
    ks[tid] = kv;
  }
  __syncthreads();
  n0 = n1 = n2 = 0.f;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    n0 += norms[0][i];
    n1 += norms[1][i];
    n2 += norms[2][i];
  }
  const float rq = a.scale * (a.l2norm ? rsqrtf(n0 + 1e-6f) : 1.f), rk = a.l2norm ? rsqrtf(n1 + 1e-6f) : 1.f;
  float4 mk = make_float4(0.f, 0.f, 0.f, 0.f), mq = mk;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float kk = ks[r * GROUPS + grp], qq = qs[r * GROUPS + grp];
    mk.x += s[r].x * kk; mk.y += s[r].y * kk; mk.z += s[r].z * kk; mk.w += s[r].w * kk;
    mq.x += s[r].x * qq; mq.y += s[r].y * qq; mq.z += s[r].z * qq; mq.w += s[r].w * qq;
  }
#pragma unroll
  for (int i = CT; i < 32; i <<= 1) {
    mk.x += __shfl_xor_sync(0xffffffffu, mk.x, i); mk.y += __shfl_xor_sync(0xffffffffu, mk.y, i);
    mk.z += __shfl_xor_sync(0xffffffffu, mk.z, i); mk.w += __shfl_xor_sync(0xffffffffu, mk.w, i);
    mq.x += __shfl_xor_sync(0xffffffffu, mq.x, i); mq.y += __shfl_xor_sync(0xffffffffu, mq.y, i);
    mq.z += __shfl_xor_sync(0xffffffffu, mq.z, i); mq.w += __shfl_xor_sync(0xffffffffu, mq.w, i);
  }
  if (lane < CT) {
    *reinterpret_cast<float4*>(&part[0][warp][col]) = mk;
    *reinterpret_cast<float4*>(&part[1][warp][col]) = mq;
  }
  __syncthreads();
  mk = mq = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    const float4 x = *reinterpret_cast<const float4*>(&part[0][i][col]);
    mk.x += x.x; mk.y += x.y; mk.z += x.z; mk.w += x.w;
  }
  const float decay = __expf(a.g[static_cast<long long>(b) * a.Hv + h]), beta = a.beta[static_cast<long long>(b) * a.Hv + h];
  const bf16* v = static_cast<const bf16*>(a.v) + b * a.v_ts + h * a.v_hs + vb * COLS + col;
  float u[4];
  const float m[4] = {mk.x, mk.y, mk.z, mk.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = beta * (__bfloat162float(v[j]) - decay * rk * m[j]);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float kk = rk * ks[r * GROUPS + grp];
    s[r].x = decay * s[r].x + kk * u[0];
    s[r].y = decay * s[r].y + kk * u[1];
    s[r].z = decay * s[r].z + kk * u[2];
    s[r].w = decay * s[r].w + kk * u[3];
    S[(r * GROUPS + grp) * ld] = s[r];
  }
  if (grp == 0) {
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(&part[1][i][col]);
      mq.x += x.x; mq.y += x.y; mq.z += x.z; mq.w += x.w;
    }
    const float kq = rq * rk * n2;
    o[col] = __float2bfloat16(decay * rq * mq.x + kq * u[0]);
    o[col + 1] = __float2bfloat16(decay * rq * mq.y + kq * u[1]);
    o[col + 2] = __float2bfloat16(decay * rq * mq.z + kq * u[2]);
    o[col + 3] = __float2bfloat16(decay * rq * mq.w + kq * u[3]);
  }
}

template <int DK>
int launch(const DeltaStepArgs& a, cudaStream_t s) {
  const long long heads = static_cast<long long>(a.B) * a.Hv;
  // 32 columns a block, 128-byte pieces of a row, while 64 leave multiprocessors with less than two blocks; else 64.
  const int cols = heads * (a.dv / 64) < 2 * sm_count() ? 32 : 64;
  const long long grid = heads * (a.dv / cols);
  if (grid > INT32_MAX) return -2;
  if (cols == 32) delta_step_kernel<DK, 32><<<static_cast<unsigned>(grid), THREADS, 0, s>>>(a);
  else delta_step_kernel<DK, 64><<<static_cast<unsigned>(grid), THREADS, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

int delta_step(const DeltaStepArgs& a, cudaStream_t s) {
  if (a.dv % 64 != 0) return -1;
  if (a.B == 0) return 0;
  if (a.dk == 64) return launch<64>(a, s);
  if (a.dk == 128) return launch<128>(a, s);
  return -1;
}

}  // namespace lf
