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
// Bound by memory. D / 16 lanes hold a head. A lane holds both elements of its rotated pairs (eight neighbours of each
// half, 16 bytes at a time; 16 neighbours behind the rotated span), so the rotation stays in the lane. A block takes
// either query heads or key heads, so that norm weight, their gradient and the pairs' factors stay in registers, and lays
// (token, head) out so that a lane keeps one token, hence its cosines, for up to eight heads. What a lane will work on is
// copied ahead, over the end of its turn too, into its own places in shared memory, so that nobody waits for anybody. The
// value (and gate) heads of the packed row are not touched forward; backward copies their gradients into the packed
// gradient, which is so written in one pass.
// 8192 tokens, 4 x 8 heads of 128: forward 41 us (3.7 TB/s), backward 74 us (3.3 TB/s); 4099 tokens, gated 2 x 16 heads of
// 256: 36 us (4.0 TB/s), backward 78 us (4.6 TB/s). Both issue every second cycle; what is left is the wait for the
// angles at each turn and the uneven last turn.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "device_info.h"
#include "elementwise.h"

namespace lf {
namespace {

using bf16 = __nv_bfloat16;
constexpr int THREADS = 256;
constexpr int STAGES = 4;       // heads of a lane under way or worked on
constexpr int ROT = THREADS * 8;  // (token, angle) pairs of a block's turn: heads at once x at most 8 LANES

// Two fp32 values in one register pair, worked on by one instruction.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 two(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 parts(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator-(F2 a, F2 b) {
  F2 r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum(F2 a) {
  const float2 p = parts(a);
  return p.x + p.y;
}
__device__ __forceinline__ float lo_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t narrow2(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cos / sin of `tokens` tokens from t0 into shared memory. The angle is a fraction of a turn, so the fast sine and cosine
// are off by 2^-21 of one at most, where the results are rounded to 2^-8.
template <int B>  // angles of a thread whose positions are fetched together
__device__ __forceinline__ void make_rotation(const QkNormRopeArgs& a, long long t0, int tokens, float* cs, float* sn) {
  const int half = a.rot_dim >> 1, dt = THREADS / half, df = THREADS - dt * half;
  int tk = threadIdx.x / half, f = threadIdx.x - tk * half;
  bool wrong = false;
  for (int i = threadIdx.x; tk < tokens; i += B * THREADS) {
    double ang[B];
    bool in[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const long long t = t0 + tk;
      in[j] = tk < tokens;
      ang[j] = 0.0;
      if (in[j] && t < a.T) {  // lanes of tokens behind the last work on zeros
        if (a.freqs) {
          const long long row = a.pos ? a.pos[t] : t;
          if (row >= 0 && row < a.freq_rows) ang[j] = a.freqs[row * half + f];
          else wrong = true;
        } else {
          const int ax = a.axis ? a.axis[f] : 0;
          if (ax >= 0 && ax < a.axes) ang[j] = static_cast<double>(a.pos[static_cast<long long>(ax) * a.T + t]) * static_cast<double>(a.inv_freq[f]);
          else wrong = true;
        }
      }
      tk += dt;
      f += df;
      if (f >= half) {
        f -= half;
        ++tk;
      }
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (!in[j]) continue;
      const double turns = ang[j] * 0.15915494309189533577;
      float s, c;
      __sincosf(static_cast<float>((turns - rint(turns)) * 6.283185307179586477), &s, &c);
      cs[i + j * THREADS] = c * a.mscale;
      sn[i + j * THREADS] = s * a.mscale;
    }
  }
  if (wrong) *a.status = 7;
}

__device__ __forceinline__ void make_rotation(const QkNormRopeArgs& a, long long t0, int tokens, float* cs, float* sn) {
  if (tokens * (a.rot_dim >> 1) <= THREADS) make_rotation<1>(a, t0, tokens, cs, sn);
  else make_rotation<4>(a, t0, tokens, cs, sn);
}

// How a lane's 16 elements lie in a head.
enum Mode {
  PAIRS,   // 16 neighbours, neighbours are pairs
  HALVES,  // eight neighbours of each half of the span; rot_dim % 16 == 0
  QUADS    // four and four of each half, for the other spans
};

// Four groups of four, in the order of memory for PAIRS; else the first halves of the pairs, then the second.
template <int MODE>
struct Place {
  int e[4], f0;  // f0: the angle of the lane's first pair
  bool in[2];    // whether pairs 0 .. 3 and 4 .. 7 rotate
  __device__ __forceinline__ Place(int rot_dim, int hl) {
    const int half = rot_dim >> 1;
    f0 = 8 * hl;
    if (MODE == PAIRS) {
      for (int i = 0; i < 4; ++i) e[i] = 16 * hl + 4 * i;
      in[0] = e[0] < rot_dim;
      in[1] = e[2] < rot_dim;
    } else if (MODE == HALVES) {
      in[0] = in[1] = f0 < half;
      e[0] = in[0] ? f0 : 16 * hl;  // behind the span: rot_dim + 16 (hl - half / 8)
      e[2] = in[0] ? half + f0 : 16 * hl + 8;
      e[1] = e[0] + 4;
      e[3] = e[2] + 4;
    } else {
      for (int s = 0; s < 2; ++s) {
        const int p = f0 + 4 * s;
        in[s] = p < half;
        e[s] = in[s] ? p : 2 * p;
        e[s + 2] = in[s] ? half + p : 2 * p + 4;
      }
    }
  }
};

struct Raw {
  uint4 a, b;
};
template <int MODE>
__device__ __forceinline__ Raw load(const bf16* p, const Place<MODE>& pl) {
  Raw r;
  if (MODE == QUADS) {
    const uint2 v0 = *reinterpret_cast<const uint2*>(p + pl.e[0]), v1 = *reinterpret_cast<const uint2*>(p + pl.e[1]);
    const uint2 v2 = *reinterpret_cast<const uint2*>(p + pl.e[2]), v3 = *reinterpret_cast<const uint2*>(p + pl.e[3]);
    r.a = make_uint4(v0.x, v0.y, v1.x, v1.y);
    r.b = make_uint4(v2.x, v2.y, v3.x, v3.y);
  } else {
    r.a = *reinterpret_cast<const uint4*>(p + pl.e[0]);
    r.b = *reinterpret_cast<const uint4*>(p + pl.e[2]);
  }
  return r;
}
template <int MODE>
__device__ __forceinline__ void store(bf16* p, const Place<MODE>& pl, const Raw& r) {
  if (MODE == QUADS) {
    *reinterpret_cast<uint2*>(p + pl.e[0]) = make_uint2(r.a.x, r.a.y);
    *reinterpret_cast<uint2*>(p + pl.e[1]) = make_uint2(r.a.z, r.a.w);
    *reinterpret_cast<uint2*>(p + pl.e[2]) = make_uint2(r.b.x, r.b.y);
    *reinterpret_cast<uint2*>(p + pl.e[3]) = make_uint2(r.b.z, r.b.w);
  } else {
    *reinterpret_cast<uint4*>(p + pl.e[0]) = r.a;
    *reinterpret_cast<uint4*>(p + pl.e[2]) = r.b;
  }
}
// The same, to come: into the thread's own 32 bytes (THREADS apart by 16) of shared memory; zeros where it is not `ok`.
template <int BYTES>
__device__ __forceinline__ void copy_ahead(uint32_t d, const void* src, bool ok) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(ok ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d), "l"(src), "r"(ok ? 8 : 0) : "memory");
}
template <int MODE>
__device__ __forceinline__ void load_ahead(uint32_t mine, const bf16* p, const Place<MODE>& pl, bool ok) {
  if (MODE == QUADS) {
    copy_ahead<8>(mine, p + pl.e[0], ok);
    copy_ahead<8>(mine + 8, p + pl.e[1], ok);
    copy_ahead<8>(mine + THREADS * 16, p + pl.e[2], ok);
    copy_ahead<8>(mine + THREADS * 16 + 8, p + pl.e[3], ok);
  } else {
    copy_ahead<16>(mine, p + pl.e[0], ok);
    copy_ahead<16>(mine + THREADS * 16, p + pl.e[2], ok);
  }
}
__device__ __forceinline__ Raw taken(const uint4* mine) { return Raw{mine[0], mine[THREADS]}; }
// Pair j of the lane is (f[j], f[j + 8]), two neighbouring j in one F2.
template <int MODE>
__device__ __forceinline__ void widen(const Raw& r, F2 (&f)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (MODE == PAIRS) {
      f[i] = two(lo_half(w[2 * i]), lo_half(w[2 * i + 1]));
      f[i + 4] = two(hi_half(w[2 * i]), hi_half(w[2 * i + 1]));
    } else {
      f[i] = two(lo_half(w[i]), hi_half(w[i]));
      f[i + 4] = two(lo_half(w[i + 4]), hi_half(w[i + 4]));
    }
  }
}
template <int MODE>
__device__ __forceinline__ Raw narrow(const F2 (&f)[8]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = parts(f[i]), y = parts(f[i + 4]);
    if (MODE == PAIRS) {
      w[2 * i] = narrow2(x.x, y.x);
      w[2 * i + 1] = narrow2(x.y, y.y);
    } else {
      w[i] = narrow2(x.x, x.y);
      w[i + 4] = narrow2(y.x, y.y);
    }
  }
  return Raw{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
}

struct Rotation {
  F2 c[4], s[4];
};
template <int MODE>
__device__ __forceinline__ Rotation rotation_of(const Place<MODE>& p, const float* cs, const float* sn) {
  Rotation r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = p.in[i >> 1];
    const float2 c = in ? *reinterpret_cast<const float2*>(cs + p.f0 + 2 * i) : make_float2(1.f, 1.f);
    const float2 s = in ? *reinterpret_cast<const float2*>(sn + p.f0 + 2 * i) : make_float2(0.f, 0.f);
    r.c[i] = two(c.x, c.y);
    r.s[i] = two(s.x, s.y);
  }
  return r;
}
template <bool BACK>
__device__ __forceinline__ void rotate(F2 (&f)[8], const Rotation& r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 x = f[i], y = f[i + 4];
    f[i] = BACK ? fma2(x, r.c[i], y * r.s[i]) : x * r.c[i] - y * r.s[i];
    f[i + 4] = BACK ? y * r.c[i] - x * r.s[i] : fma2(y, r.c[i], x * r.s[i]);
  }
}

template <int MODE>
__device__ __forceinline__ void weights(const bf16* p, const Place<MODE>& pl, float offset, F2 (&w)[8]) {
  widen<MODE>(load(p, pl), w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = parts(w[i]);
    w[i] = two(v.x + offset, v.y + offset);
  }
}

// The heads of one kind: `per` of a group from head `base` of its `P`, `count` of a token. A block's turn is `tokens`
// tokens with 2^lg lanes' worth of heads of each at a time.
struct Part {
  int per, base, count, lg, tokens, block, blocks;
  const bf16* w;
  template <int LANES>
  __device__ __forceinline__ static Part of(const QkNormRopeArgs& a) {
    constexpr int HEADS = THREADS / LANES;
    Part p;
    const bool q = static_cast<int>(blockIdx.x) < a.q_blocks;
    p.per = q ? a.R : 1;
    p.base = q ? 0 : a.P - 2;
    p.count = a.G * p.per;
    p.w = static_cast<const bf16*>(q ? a.qw : a.kw);
    p.lg = q ? a.q_lg : a.k_lg;
    p.tokens = HEADS >> p.lg;
    p.block = q ? blockIdx.x : blockIdx.x - a.q_blocks;
    p.blocks = q ? a.q_blocks : gridDim.x - a.q_blocks;
    return p;
  }
};
// The heads of a lane, 2^lg apart, without a division each.
struct Head {
  int h, r;  // its number among the token's, and in its group
  int off;   // where it lies in the packed row, in elements from the first of its kind
};
struct Stride {
  Head first;
  int per, dh, dr, doff, wrap;
  __device__ __forceinline__ Stride(const Part& p, int start, int P, int D) : per(p.per), dh(1 << p.lg) {
    const int g0 = start / per, dg = dh / per;
    wrap = (P - per) * D;
    first = {start, start - g0 * per, start * D + g0 * wrap};
    dr = dh - dg * per;
    doff = dh * D + dg * wrap;
  }
  __device__ __forceinline__ void next(Head& x) const {
    x.h += dh;
    x.r += dr;
    x.off += doff;
    if (x.r >= per) {
      x.r -= per;
      x.off += wrap;
    }
  }
};

// A lane's walk over its heads and on to its next tokens, with the rows of up to two tensors.
struct Walk {
  int left, n;  // tokens up to the last one from here on; the turn
  Head at;
  const bf16 *x, *g;
  __device__ __forceinline__ Walk(const QkNormRopeArgs& a, const Part& p, int tk, const Head& first, const bf16* x0, long long xs, const bf16* g0, long long gs) {
    const int t = p.block * p.tokens + tk;
    left = static_cast<int>(a.T) - t;
    n = 0;
    at = first;
    x = x0 + t * xs;
    g = g0 + t * gs;
  }
  __device__ __forceinline__ void next(const Part& p, const Stride& st, int turns, long long xgo, long long ggo) {
    st.next(at);
    if (++n == turns) {
      n = 0;
      at = st.first;
      left -= p.blocks * p.tokens;
      x += xgo;
      g += ggo;
    }
  }
};

struct FwdSmem {
  float cs[2][ROT], sn[2][ROT];
  uint4 x[STAGES][2][THREADS];
};
struct BwdSmem {
  float cs[2][ROT], sn[2][ROT];
  union {
    uint4 in[STAGES][4][THREADS];  // dy, x
    float red[THREADS * 16];
  };
};

template <int LANES, int MODE>
__global__ void __launch_bounds__(THREADS, 3)
qk_fwd_kernel(const QkNormRopeArgs a) {
  constexpr int D = LANES * 16;
  extern __shared__ __align__(16) unsigned char smem[];
  FwdSmem& sm = *reinterpret_cast<FwdSmem*>(smem);
  const Part p = Part::of<LANES>(a);
  const int hl = threadIdx.x % LANES, slot = threadIdx.x / LANES, tk = slot >> p.lg, step = 1 << p.lg, half = a.rot_dim >> 1;
  const Place<MODE> pl(a.rot_dim, hl);
  const Stride st(p, slot & (step - 1), a.P, D);
  const long long go = static_cast<long long>(p.blocks) * p.tokens;
  // every lane of a warp makes the same number of turns: the sums over a head need them all
  const int turns = (p.count + step - 1) >> p.lg;
  const bf16* const x = static_cast<const bf16*>(a.x) + p.base * D;
  Walk ahead(a, p, tk, st.first, x, a.x_ts, x, 0);
  const uint32_t mine = static_cast<uint32_t>(__cvta_generic_to_shared(&sm.x[0][0][threadIdx.x]));
  auto fetch = [&](unsigned stage) {
    const bool ok = ahead.left > 0 && ahead.at.h < p.count;
    load_ahead(mine + stage * sizeof(sm.x[0]), ok ? ahead.x + ahead.at.off : x, pl, ok);
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead.next(p, st, turns, go * a.x_ts, 0);
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);
  F2 w[8];
  weights(p.w, pl, a.w_offset, w);
  bf16* const out = static_cast<bf16*>(p.base == 0 ? a.q : a.k);
  unsigned stage = 0, buf = 0;
  for (long long t0 = static_cast<long long>(p.block) * p.tokens; t0 < a.T; t0 += go) {
    const long long t = t0 + tk;
    const bool live = t < a.T;
    bf16* dst = out + t * p.count * D;
    make_rotation(a, t0, p.tokens, sm.cs[buf], sm.sn[buf]);
    __syncthreads();
    const Rotation rot = rotation_of(pl, sm.cs[buf] + tk * half, sm.sn[buf] + tk * half);
    buf ^= 1;
    Head at = st.first;
#pragma unroll 1
    for (int n = 0; n < turns; ++n) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      F2 f[8];
      widen<MODE>(taken(&sm.x[stage][0][threadIdx.x]), f);
      fetch((stage + STAGES - 1) % STAGES);
      stage = (stage + 1u) % STAGES;
      F2 ss = two(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fma2(f[j], f[j], ss);
      const float rstd = rsqrtf(head_sum<LANES>(sum(ss)) * (1.f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * two(rstd, rstd) * w[j];
      rotate<false>(f, rot);
      if (live && at.h < p.count) store(dst + at.h * D, pl, narrow<MODE>(f));
      st.next(at);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int LANES, int MODE>
__global__ void __launch_bounds__(THREADS, 2)
qk_bwd_kernel(const QkNormRopeArgs a) {
  constexpr int D = LANES * 16, HEADS = THREADS / LANES;
  extern __shared__ __align__(16) unsigned char smem[];
  BwdSmem& sm = *reinterpret_cast<BwdSmem*>(smem);
  const Part p = Part::of<LANES>(a);
  const int hl = threadIdx.x % LANES, slot = threadIdx.x / LANES, tk = slot >> p.lg, step = 1 << p.lg, half = a.rot_dim >> 1;
  const Place<MODE> pl(a.rot_dim, hl);
  const Stride st(p, slot & (step - 1), a.P, D);
  const long long go = static_cast<long long>(p.blocks) * p.tokens;
  const int turns = (p.count + step - 1) >> p.lg;
  const bool q = p.base == 0;
  const bf16* const x = static_cast<const bf16*>(a.x) + p.base * D;
  const bf16* const grad = static_cast<const bf16*>(q ? a.dq : a.dk);
  // heads whose gradient is copied: the gate's beside the queries, the values beside the keys
  const bf16* const copy = static_cast<const bf16*>(q ? a.dgate : a.dv);
  const int copy_base = q ? a.R : a.P - 1;
  Walk ahead(a, p, tk, st.first, x, a.x_ts, grad, p.count * D);
  const uint32_t own = static_cast<uint32_t>(__cvta_generic_to_shared(&sm.in[0][0][threadIdx.x]));
  auto fetch = [&](unsigned stage) {
    const bool ok = ahead.left > 0 && ahead.at.h < p.count;
    load_ahead(own + stage * sizeof(sm.in[0]), ok ? ahead.g + ahead.at.h * D : grad, pl, ok);
    load_ahead(own + stage * sizeof(sm.in[0]) + sizeof(sm.in[0][0]) * 2, ok ? ahead.x + ahead.at.off : x, pl, ok);
    asm volatile("cp.async.commit_group;" ::: "memory");
    ahead.next(p, st, turns, go * a.x_ts, go * p.count * D);
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);
  F2 w[8], dw[8];
  weights(p.w, pl, a.w_offset, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[j] = two(0.f, 0.f);
  unsigned stage = 0, buf = 0;
  for (long long t0 = static_cast<long long>(p.block) * p.tokens; t0 < a.T; t0 += go) {
    const long long t = t0 + tk;
    const bool live = t < a.T;
    bf16* dxrow = static_cast<bf16*>(a.dx) + t * a.G * a.P * D;
    const bf16* crow = copy + t * p.count * D + 8 * hl;
    make_rotation(a, t0, p.tokens, sm.cs[buf], sm.sn[buf]);
    __syncthreads();
    const Rotation rot = rotation_of(pl, sm.cs[buf] + tk * half, sm.sn[buf] + tk * half);
    buf ^= 1;
    Head at = st.first;
#pragma unroll 1
    for (int n = 0; n < turns; ++n) {
      uint4 v0, v1;
      const bool mine = live && at.h < p.count;
      if (copy && mine) {
        const bf16* c = crow + at.h * D;
        v0 = *reinterpret_cast<const uint4*>(c);
        v1 = *reinterpret_cast<const uint4*>(c + D / 2);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      F2 d[8], x[8];
      widen<MODE>(taken(&sm.in[stage][0][threadIdx.x]), d);
      widen<MODE>(taken(&sm.in[stage][2][threadIdx.x]), x);
      fetch((stage + STAGES - 1) % STAGES);
      stage = (stage + 1u) % STAGES;
      rotate<true>(d, rot);
      // the two sums over the head: x . x and d w . x
      F2 ss = two(0.f, 0.f), dots = ss;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ss = fma2(x[j], x[j], ss);
        dots = fma2(d[j] * x[j], w[j], dots);
      }
      const float s = head_sum<LANES>(sum(ss)), dot = head_sum<LANES>(sum(dots));
      // a lane without a head works on zeros, whose root is zero when eps is: nothing of it may reach dw
      const float rstd = mine ? rsqrtf(s * (1.f / D) + a.eps) : 0.f, m = dot * rstd * rstd * rstd * (1.f / D);
      const F2 rr = two(rstd, rstd), mm = two(m, m);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        d[j] = d[j] * rr;
        dw[j] = fma2(d[j], x[j], dw[j]);
        d[j] = d[j] * w[j] - x[j] * mm;
      }
      if (mine) {
        bf16* o = dxrow + at.off;
        store(o + p.base * D, pl, narrow<MODE>(d));
        if (copy) {
          *reinterpret_cast<uint4*>(o + copy_base * D + 8 * hl) = v0;
          *reinterpret_cast<uint4*>(o + copy_base * D + 8 * hl + D / 2) = v1;
        }
      }
      st.next(at);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float (*red)[D] = reinterpret_cast<float (*)[D]>(sm.red);
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // pairs 2 (i % 4) and the next, first or second halves
    const float2 v = parts(dw[i]);
    const int j = 2 * (i & 3), y = i >> 2;
    const int at = MODE == PAIRS ? pl.e[0] + 2 * j + y : pl.e[2 * y + (j >> 2)] + (j & 3);
    red[slot][at] = v.x;
    red[slot][at + (MODE == PAIRS ? 2 : 1)] = v.y;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < D; c += THREADS) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < HEADS; ++i) s += red[i][c];
    a.partial[static_cast<long long>(blockIdx.x) * D + c] = s;
  }
}

// dw = sum over the blocks of its kind of partial[b, c] in a fixed order: a block per 32 columns, 32 rows of threads.
__global__ void qk_dw_kernel(const float* __restrict__ partial, int q_blocks, int blocks, int D, bf16* __restrict__ dqw, bf16* __restrict__ dkw) {
  __shared__ float red[32][33];
  const bool q = blockIdx.x * 32 < D;
  const int c0 = blockIdx.x * 32 - (q ? 0 : D), end = q ? q_blocks : blocks;
  float s = 0.f;
#pragma unroll 8
  for (int b = (q ? 0 : q_blocks) + threadIdx.y; b < end; b += 32) s += partial[static_cast<long long>(b) * D + c0 + threadIdx.x];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = red[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x == 0) (q ? dqw : dkw)[c0 + threadIdx.y] = __float2bfloat16(s);
}

// How a launch is laid out; returns its blocks. A lane keeps up to eight heads of its token, which makes the angles cheap
// (8192 tokens of 4 x 8 heads of 128, forward + backward: 116 us with two, 125 with four, 115 with eight), and fewer while the
// tokens do not give every block two turns. The two kinds share the blocks in proportion to their work (a head's elements,
// and twice as much for an angle), and none has more than the tokens ask for.
int lay_out(QkNormRopeArgs& a, int room) {
  const int heads = THREADS / (a.D / 16);
  auto at_once = [&](int count, int keep) {  // log2 of a token's heads that a block works on at once
    int lg = 0;
    while (((2 * keep) << lg <= count || (heads >> lg > 2 * keep && 1 << lg < count)) && 2 << lg <= heads) ++lg;
    return lg;
  };
  auto turns = [&](int lg) { return (a.T + (heads >> lg) - 1) / (heads >> lg); };
  for (int keep = 8; keep > 0; keep >>= 1) {
    a.q_lg = at_once(a.G * a.R, keep);
    a.k_lg = at_once(a.G, keep);
    if (turns(a.q_lg) + turns(a.k_lg) >= 2 * room) break;
  }
  const long long q = turns(a.q_lg), k = turns(a.k_lg);
  const double wq = static_cast<double>(a.G) * a.R * a.D + 2.0 * a.rot_dim, wk = static_cast<double>(a.G) * a.D + 2.0 * a.rot_dim;
  int ks = static_cast<int>(room * (wk / (wq + wk)) + 0.5);
  ks = static_cast<int>(k < ks ? k : ks > 1 ? ks : 1);
  a.q_blocks = static_cast<int>(q < room - ks ? q : room - ks);
  return a.q_blocks + ks;
}

template <auto KERNEL>
int launch(size_t bytes, const QkNormRopeArgs& a, int grid, cudaStream_t s) {
  static std::atomic<uint64_t> allowed{0};
  if (!allow_smem(KERNEL, bytes, allowed)) return -3;
  KERNEL<<<static_cast<unsigned>(grid), THREADS, bytes, s>>>(a);
  return 0;
}
template <int LANES>
int launch_fwd(const QkNormRopeArgs& a, int grid, cudaStream_t s) {
  if (a.interleaved) return launch<qk_fwd_kernel<LANES, PAIRS>>(sizeof(FwdSmem), a, grid, s);
  if (a.rot_dim % 16 == 0) return launch<qk_fwd_kernel<LANES, HALVES>>(sizeof(FwdSmem), a, grid, s);
  return launch<qk_fwd_kernel<LANES, QUADS>>(sizeof(FwdSmem), a, grid, s);
}
template <int LANES>
int launch_bwd(const QkNormRopeArgs& a, int grid, cudaStream_t s) {
  if (a.interleaved) return launch<qk_bwd_kernel<LANES, PAIRS>>(sizeof(BwdSmem), a, grid, s);
  if (a.rot_dim % 16 == 0) return launch<qk_bwd_kernel<LANES, HALVES>>(sizeof(BwdSmem), a, grid, s);
  return launch<qk_bwd_kernel<LANES, QUADS>>(sizeof(BwdSmem), a, grid, s);
}
bool covered(const QkNormRopeArgs& a) { return (a.D == 64 || a.D == 128 || a.D == 256) && a.rot_dim <= a.D; }

}  // namespace

int qk_norm_rope_bwd_grid(QkNormRopeArgs& a) {
  return a.T == 0 ? 0 : lay_out(a, sm_count() * 2);
}

int qk_norm_rope_fwd(QkNormRopeArgs& a, cudaStream_t s) {
  if (!covered(a)) return -1;
  if (a.T > INT32_MAX / 2) return -2;
  if (a.T == 0) return 0;
  const int blocks = lay_out(a, sm_count() * 3);
  const int rc = a.D == 64 ? launch_fwd<4>(a, blocks, s) : a.D == 128 ? launch_fwd<8>(a, blocks, s) : launch_fwd<16>(a, blocks, s);
  if (rc != 0) return rc;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int qk_norm_rope_bwd(QkNormRopeArgs& a, cudaStream_t s) {
  if (!covered(a)) return -1;
  if (a.T > INT32_MAX / 2) return -2;
  const int grid = qk_norm_rope_bwd_grid(a);
  if (grid > 0) {
    const int rc = a.D == 64 ? launch_bwd<4>(a, grid, s) : a.D == 128 ? launch_bwd<8>(a, grid, s) : launch_bwd<16>(a, grid, s);
    if (rc != 0) return rc;
  }
  qk_dw_kernel<<<2 * a.D / 32, dim3(32, 32), 0, s>>>(a.partial, a.q_blocks, grid, a.D, static_cast<bf16*>(a.dqw), static_cast<bf16*>(a.dkw));
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace lf
