// Parts that the kernels of the gated delta rule share: the factor block of a chunk, the plan of the sequences, the split of
// fp32 operands into two bf16 parts, and the barriers between the warps of a block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "device_info.h"
#include "linear_attn.h"

namespace lf {
namespace delta {

using bf16 = __nv_bfloat16;
constexpr int C = DELTA_CHUNK;

// Rows of a chunk's factor block, 64 floats each.
enum { V_YK = 0, V_BETA, V_OQ, V_SU, V_GHI, V_GLO, V_QS, V_RK, V_END, V_PD, V_RQ };  // V_PD: diagonal of P
constexpr int ROW_DOTS = 3;  // sums over the columns that the backward chain leaves for every token, per unit: see there
constexpr int SEQ_ROWS = V_PD + 1;  // rows that the kernels along the sequence read

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void cp16(void* dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
// With the remainder of the second rounding too: x and y but for 2^-26.
__device__ __forceinline__ void split3(float x, float y, uint32_t& hi, uint32_t& lo, uint32_t& rest) {
  asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
  x -= lo_half(hi);
  y -= hi_half(hi);
  lo = pack2(x, y);
  rest = pack2(x - lo_half(lo), y - hi_half(lo));
}
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

// W_ii = qs_i rk_i do_i.u_i, without the decay that the rest of W carries: the largest part of dq and dk in heads that forget
// at once. From the sums of the backward chain, so that it is as exact as U.
__device__ __forceinline__ float w_diagonal(const DeltaArgs& a, long long rec, int i, const float* vec) {
  const float* rd = a.rowdots + (rec * (a.dv / 16) * ROW_DOTS + 2) * 64 + i;
  float s = 0.f;
#pragma unroll 8
  for (int v = 0; v < a.dv / 16; ++v) s += rd[v * ROW_DOTS * 64];
  return vec[V_QS * 64 + i] * vec[V_RK * 64 + i] * s;
}

// Barriers between the warps of a block and of a buffer's copies. They complete in every chunk, so a wait ends unless the
// kernel is wrong; after a limit far above any chunk's time it reports and goes on.
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {  // whole warp; what its lanes wrote is seen behind the wait
  __syncwarp();
  if ((threadIdx.x & 31) == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ void bar_wait(uint64_t* b, uint32_t parity, int* status) {
  uint32_t done = 0;
  for (int i = 0; i < (1 << 22); ++i) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_addr(b)), "r"(parity) : "memory");
    if (done) return;
  }
  *status = 1;
}

}  // namespace delta
}  // namespace lf
