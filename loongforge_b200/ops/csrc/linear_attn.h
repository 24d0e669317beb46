// Host launchers of the linear-attention kernels: the gated delta rule (gated_delta_sm100.cu, gated_delta_step.cu)
// and the depthwise causal convolution in front of it (causal_conv.cu). Raw pointers + stream; strides in elements.
#pragma once
#include <cuda_runtime.h>

namespace lf {

constexpr int DELTA_CHUNK = 64;      // tokens of one chunk
constexpr int DELTA_VEC = 11 * 64;   // fp32 words of one chunk's per-token factors (see the prepare kernel)
constexpr int DELTA_AP = 4 * 64 * 72;  // bf16 words of one chunk's inverse and score matrix (high and low parts, rows of 72)
constexpr int DELTA_ROW_PAD = 8;       // bf16 behind every row of a chunk's q and k tiles

struct DeltaArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;  // bf16 [T, Hk, dk], [T, Hk, dk], [T, Hv, dv]
  long long q_ts = 0, q_hs = 0, k_ts = 0, k_hs = 0, v_ts = 0, v_hs = 0;
  const float *g = nullptr, *beta = nullptr;  // fp32 [T, Hv]
  // Sequence plan: cu [N + 1] (clamped, non-decreasing) and first chunk of every sequence [N + 1]; null = one sequence.
  const int *cu = nullptr, *cbase = nullptr;
  int N = 1, Hk = 0, Hv = 0, dk = 0, dv = 0;
  long long T = 0, NC = 0;  // NC: upper bound of the number of chunks
  float scale = 1.f;
  int l2norm = 1;
  const float* s_in = nullptr;  // [N, Hv, dk, dv] or null (zero)
  float* s_out = nullptr;       // [N, Hv, dk, dv] or null
  void *o = nullptr;            // bf16 [T, Hv, dv]
  // Kept for the backward pass (all or none), as the fragments that one warp's lanes hold, [NC, Hv, dv / 16, 4, ..., 32]:
  // what o owes to earlier tokens, the memory read at each token and U (fp32); and the state in front of every chunk (bf16
  // and the remainder of the rounding).
  void *past = nullptr, *mem = nullptr, *u = nullptr, *states = nullptr;
  void* qk = nullptr;    // bf16 [NC, Hk, 2, 64, dk + DELTA_ROW_PAD]: q and k of every chunk, rows behind its end zero
  void* ap = nullptr;    // bf16 [NC, Hv, DELTA_AP]
  float* vec = nullptr;  // fp32 [NC, Hv, DELTA_VEC]
  // backward
  const void* dout = nullptr;   // bf16 [T, Hv, dv], contiguous
  const float* ds_out = nullptr;  // gradient of s_out or null
  float* ds_in = nullptr;         // gradient of s_in or null
  void* dstates = nullptr;      // the gradients of the states behind every chunk, as `states`
  void* dv_lo = nullptr;        // what the rounding of dv_ left, in bf16: fragments of half the size of `u`
  float* rowdots = nullptr;     // fp32 [NC, Hv, dv / 16, 3, 64]
  float* sdots = nullptr;       // fp32 [NC, Hv, dv / 16, 4]
  void *dq = nullptr, *dkey = nullptr, *dv_ = nullptr;  // bf16, contiguous
  float *dg = nullptr, *dbeta = nullptr;                // fp32 [T, Hv]
  int* status = nullptr;  // set when a wait runs out
};

// 0 on success; negative when the shape is not covered (dk, dv in {64, 128}).
int delta_plan(const int* cu_in, int N, long long T, int* cu, int* cbase, int* status, cudaStream_t s);
int delta_forward(const DeltaArgs& a, cudaStream_t s);
int delta_backward(const DeltaArgs& a, cudaStream_t s);
int delta_tc_dqk(const DeltaArgs& a, cudaStream_t s);  // its dq / dk for dk = dv = 128 (gated_delta_dqk_sm100.cu)
struct DeltaStepArgs {
  const void *q = nullptr, *k = nullptr, *v = nullptr;  // bf16 [B, Hk, dk], [B, Hk, dk], [B, Hv, dv]
  long long q_ts = 0, q_hs = 0, k_ts = 0, k_hs = 0, v_ts = 0, v_hs = 0;
  const float *g = nullptr, *beta = nullptr;  // [B, Hv]
  float* state = nullptr;                     // [slots, Hv, dk, dv], updated in place
  const int* index = nullptr;                 // [B] slot of each row, negative = no row; null = row b uses slot b
  void* o = nullptr;                          // bf16 [B, Hv, dv]
  int B = 0, Hk = 0, Hv = 0, dk = 0, dv = 0;
  long long slots = 0;
  float scale = 1.f;
  int l2norm = 1;
  int* status = nullptr;
};
int delta_step(const DeltaStepArgs& a, cudaStream_t s);

struct ConvArgs {
  const void* x = nullptr;  // bf16 [T, C], row stride x_ts
  long long x_ts = 0;
  const void *w = nullptr, *bias = nullptr;  // bf16 [C, K], [C] or null
  const int* cu = nullptr;                   // [N + 1] or null
  int N = 1, C = 0, K = 0, silu = 1;
  long long T = 0;
  void* y = nullptr;            // bf16 [T, C]
  const void* dy = nullptr;     // bf16 [T, C]
  void* dx = nullptr;           // bf16 [T, C]
  float* partial = nullptr;     // fp32 [conv_blocks(T, C), K + 1, C]
  void *dw = nullptr, *db = nullptr;  // bf16
};
int conv_blocks(long long T, int C);
int conv_fwd(const ConvArgs& a, cudaStream_t s);
int conv_bwd(const ConvArgs& a, cudaStream_t s);

struct ConvStepArgs {
  const void* x = nullptr;  // bf16 [B, C], row stride x_ts
  long long x_ts = 0;
  const void *w = nullptr, *bias = nullptr;
  void* state = nullptr;       // bf16 [slots, C, K - 1], updated in place
  const int* index = nullptr;  // [B] or null
  void* y = nullptr;           // bf16 [B, C]
  int B = 0, C = 0, K = 0, silu = 1;
  long long slots = 0;
  int* status = nullptr;
};
int conv_step(const ConvStepArgs& a, cudaStream_t s);

}  // namespace lf
