// Norms of queries and keys for each head, the rotary embedding and the head-first layout
// in one pass for gfx950, and their backward.
//
//   y = x r w,  r = (mean(x^2) + eps)^-1/2 over a head's D values; then the first R
//   dimensions rotated, pair (d, d + R/2): z_d = y_d cos_d - y_(d + R/2) sin_d, and
//   z_(d + R/2) = y_(d + R/2) cos_(d + R/2) + y_d sin_(d + R/2)
//
// and back, dy the gradient behind the rotation:
//   dx = r w dy - x r^3 mean(x w dy),  dw = sum over tokens of x r dy
//
// Bound by memory: each value is read once and written once, four lanes to a head's
// row, of which each takes 8 pairs of dimensions. A thread stays with one token, whose row of the tables it reads once,
// and goes over heads, the next one's values on their way. The weights' gradients stay in registers
// until a weight row ends; a block's go to memory, and a second kernel adds those up, in order.
// Arithmetic and sums are in fp32, one rounding to the tensors' type.
//
// 4 x 4096 tokens, 14 query and 2 key heads of 64, bf16: forward 15 us (75 MB in and out, 5.1 TB/s), backward 22 and the
// weights' sums 3 (109 MB, 4.3 TB/s). One token: 3.5 us, a launch and two waits for memory.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "oal_common.hpp"
#include "oal_heads.hpp"
#include "oal_tile.hpp"

namespace oal {

namespace {

constexpr int kThr = 256;
constexpr int kTokens = kThr / 4;  // a block's tokens
constexpr int kSumThr = 1024;

typedef float f32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x8 load8(const float* p) {
  const f32x4 a = load4(p), b = load4(p + 4);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x8 load8(const uint16_t* p) {
  return __builtin_convertvector(*reinterpret_cast<const bf16x8*>(p), f32x8);
}
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x8 load8(const _Float16* p) {
  return __builtin_convertvector(*reinterpret_cast<const f16x8*>(p), f32x8);
}
__device__ __forceinline__ void store8(float* p, const f32x8& x) {
  store4(p, __builtin_shufflevector(x, x, 0, 1, 2, 3));
  store4(p + 4, __builtin_shufflevector(x, x, 4, 5, 6, 7));
}
__device__ __forceinline__ void store8(uint16_t* p, const f32x8& x) {
  *reinterpret_cast<bf16x8*>(p) = __builtin_convertvector(x, bf16x8);
}
__device__ __forceinline__ void store8(_Float16* p, const f32x8& x) {
  *reinterpret_cast<f16x8*>(p) = __builtin_convertvector(x, f16x8);
}

struct Pair {
  f32x8 lo, hi;
};

// Lane j's 8 pairs of a row's D values: the first R / 2 pairs are those that the rotation
// turns, (p, p + R / 2), the others two of the rest. With WIDE a lane's lo and hi are 8 values in a row
// each (R / 2 and (D - R) / 2 multiples of 8, rows 16-byte aligned).
template <bool WIDE>
struct Place {
  int D, R, j;
  __device__ __forceinline__ bool turned(int e) const { return 8 * j + e < R / 2; }
  __device__ __forceinline__ int lo(int e) const {
    const int p = 8 * j + e;
    return p < R / 2 ? p : R + 2 * (p - R / 2);
  }
  __device__ __forceinline__ int hi(int e) const { return lo(e) + (turned(e) ? R / 2 : WIDE ? 8 : 1); }
  // fill: what a lane's places past D hold, and (angles) the places that are not turned
  template <bool ANGLES = false, typename T>
  __device__ __forceinline__ Pair load(const T* p, float fill = 0.f) const {
    Pair x;
    if constexpr (WIDE) {
      const bool in = ANGLES ? turned(0) : lo(0) < D;
      x.lo = x.hi = fill;
      if (in) x.lo = load8(p + lo(0)), x.hi = load8(p + hi(0));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int l = lo(e), h = hi(e);
        const bool a = ANGLES ? turned(e) : l < D, b = ANGLES ? turned(e) : h < D;
        x.lo[e] = a ? get(p + (a ? l : 0)) : fill;
        x.hi[e] = b ? get(p + (b ? h : 0)) : fill;
      }
    }
    return x;
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p, const Pair& x) const {
    if constexpr (WIDE) {
      if (lo(0) < D) {
        store8(p + lo(0), x.lo);
        store8(p + hi(0), x.hi);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (lo(e) < D) put(p + lo(e), x.lo[e]);
        if (hi(e) < D) put(p + hi(e), x.hi[e]);
      }
    }
  }
};

// A sum over the four lanes of a row.
__device__ __forceinline__ float row_sum(float x) {
  x += __shfl_xor(x, 1, 64);
  return x + __shfl_xor(x, 2, 64);
}
__device__ __forceinline__ float dot(const Pair& x, const Pair& y) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) s += x.lo[e] * y.lo[e] + x.hi[e] * y.hi[e];
  return s;
}
// The reciprocal root of a row's mean square.
__device__ __forceinline__ float root(const Pair& x, const HeadsArgs& a) {
  return 1.f / sqrtf(row_sum(dot(x, x)) / a.D + a.eps);
}

template <typename T, typename P>
__device__ __forceinline__ Pair weight(const HeadsArgs& a, const P& at, const void* w, int h) {
  const size_t from = a.per_head ? (size_t)h * a.D : 0;
  if (!w) return {1.f, 1.f};
  return a.w32 ? at.load(static_cast<const float*>(w) + from) : at.load(static_cast<const T*>(w) + from);
}

// A block's tokens and heads: 64 tokens, thread t's the token t / 4, and the heads [first, last) of all
// of q, k and v. A thread keeps its token, whose row of the tables it reads once.
struct Part {
  int64_t token;
  int b, n, first, last;
  bool live;
  int64_t pos;
  __device__ __forceinline__ Part(const HeadsArgs& a, int each) {
    const int64_t i = (int64_t)blockIdx.x * kTokens + (threadIdx.x >> 2), total = (int64_t)a.B * a.N;
    live = i < total;
    token = live ? i : total - 1;
    b = (int)((uint32_t)token / (uint32_t)a.N);  // fewer than 2^30 tokens
    n = (int)(token - (int64_t)b * a.N);
    first = blockIdx.y * each;
    last = min(first + each, a.Hq + 2 * a.Hk);
    pos = a.position ? a.position[token] : n;
  }
};

// cos and sin of a position; past the tables NaN.
template <typename T, typename P>
__device__ __forceinline__ void angles(const HeadsArgs& a, const P& at, int64_t pos, Pair& cosine, Pair& sine) {
  const bool in = pos >= 0 && pos < a.table;
  const size_t from = in ? (size_t)pos * a.R : 0;
  if (a.t32) {
    cosine = at.template load<true>(static_cast<const float*>(a.cosine) + from, 1.f);
    sine = at.template load<true>(static_cast<const float*>(a.sine) + from, 0.f);
  } else {
    cosine = at.template load<true>(static_cast<const T*>(a.cosine) + from, 1.f);
    sine = at.template load<true>(static_cast<const T*>(a.sine) + from, 0.f);
  }
  if (pos >= a.table) cosine.lo = cosine.hi = __builtin_nanf("");
}

}  // namespace

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThr) void k_heads(HeadsArgs a, int each, T* __restrict__ hq, T* __restrict__ hk,
                                                T* __restrict__ hv) {
  const Part p(a, each);
  if (!p.live) return;
  const Place<WIDE> at{a.D, a.R, (int)(threadIdx.x & 3)};
  auto fetch = [&](int h) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
    const int own = is_q ? h : is_v ? h - a.Hq - a.Hk : h - a.Hq;
    return at.load(static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + p.b * (is_q ? a.qb : is_v ? a.vb : a.kb) +
                   p.n * (is_q ? a.qn : is_v ? a.vn : a.kn) + own * a.D);
  };
  Pair next = fetch(p.first), cosine, sine, w;
  angles<T>(a, at, p.pos, cosine, sine);
  for (int h = p.first; h < p.last; ++h) {
    Pair x = next;
    if (h + 1 < p.last) next = fetch(h + 1);
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hk;
    const int own = is_q ? h : is_v ? h - a.Hq - a.Hk : h - a.Hq;
    if (!is_v) {
      if (h == p.first || h == a.Hq || a.per_head) w = weight<T>(a, at, is_q ? a.qw : a.kw, own);
      const float r = root(x, a);
      const f32x8 lo = x.lo * r * w.lo, hi = x.hi * r * w.hi;
      x.lo = lo * cosine.lo - hi * sine.lo;
      x.hi = hi * cosine.hi + lo * sine.hi;
    }
    if (p.pos < 0) x.lo = x.hi = 0.f;
    at.store((is_q ? hq : is_v ? hv : hk) + (((int64_t)p.b * (is_q ? a.Hq : a.Hk) + own) * a.N + p.n) * a.D, x);
  }
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThr) void k_heads_bwd(HeadsArgs a, int each, const T* __restrict__ hq,
                                                    const T* __restrict__ hk, const T* __restrict__ hv,
                                                    T* __restrict__ dq, T* __restrict__ dk, T* __restrict__ dv,
                                                    float* __restrict__ work) {
  __shared__ alignas(16) float sums[kTokens][68];
  __shared__ float parts[kThr / 64][64];
  const Part p(a, each);
  const Place<WIDE> at{a.D, a.R, (int)(threadIdx.x & 3)};
  // a place without a token asks for nothing
  const bool there = p.live && p.pos >= 0;
  Pair cosine, sine;
  angles<T>(a, at, p.pos, cosine, sine);
  const int targets = a.per_head ? a.Hq + a.Hk : 2;
  float* const rows = work + (a.per_head ? blockIdx.x : (size_t)blockIdx.y * gridDim.x + blockIdx.x) * targets * a.D;
  // the part's heads of q or k: source x, gradients up and out, both from the projections' and the heads' first
  auto norms = [&](const T* x0, int64_t xb, int64_t xn, const void* weights, const T* up0, T* out0, int H, int from,
                   int to, int target) __attribute__((always_inline)) {
    if (from >= to) {
      if (work && !a.per_head && (int)threadIdx.x < a.D) rows[target * a.D + threadIdx.x] = 0.f;
      return;
    }
    const T* x1 = x0 + p.b * xb + p.n * xn;
    const T* up1 = up0 + ((int64_t)p.b * H * a.N + p.n) * a.D;
    T* out1 = out0 + p.token * H * a.D;
    Pair w{}, g{}, x = at.load(x1 + from * a.D), up{};
    if (up0 && there) up = at.load(up1 + (int64_t)from * a.N * a.D);
    for (int h = from; h < to; ++h) {
      Pair nx{}, nup{};
      if (h + 1 < to) {
        nx = at.load(x1 + (h + 1) * a.D);
        if (up0 && there) nup = at.load(up1 + (int64_t)(h + 1) * a.N * a.D);
      }
      if (h == from || a.per_head) w = weight<T>(a, at, weights, h);
      const float r = root(x, a);
      Pair y;
      y.lo = up.lo * cosine.lo + up.hi * sine.hi;
      y.hi = up.hi * cosine.hi - up.lo * sine.lo;
      x.lo *= r, x.hi *= r;
      if (there) g.lo += x.lo * y.lo, g.hi += x.hi * y.hi;
      y.lo *= w.lo, y.hi *= w.hi;
      const float mean = row_sum(dot(x, y)) / a.D;
      up.lo = r * (y.lo - x.lo * mean), up.hi = r * (y.hi - x.hi * mean);
      if (!there) up = Pair{};
      if (out0 && p.live) at.store(out1 + h * a.D, up);
      x = nx, up = nup;
      if (work && (a.per_head || h + 1 == to)) {
        // the block's sum of a weight row's gradient, tokens in order
        const int d = threadIdx.x & 63, part = threadIdx.x >> 6;
        at.store(sums[threadIdx.x >> 2], g);
        g = Pair{};
        __syncthreads();
        float s = 0.f;
        if (d < a.D)
          for (int i = 0; i < kTokens / 4; ++i) s += sums[part * (kTokens / 4) + i][d];
        parts[part][d] = s;
        __syncthreads();
        if (part == 0 && d < a.D)
          rows[(target + (a.per_head ? h : 0)) * a.D + d] = (parts[0][d] + parts[1][d]) + (parts[2][d] + parts[3][d]);
      }
    }
  };
  const int k0 = a.Hq, v0 = a.Hq + a.Hk;
  norms(static_cast<const T*>(a.q), a.qb, a.qn, a.qw, hq, dq, a.Hq, p.first, min(p.last, k0), 0);
  norms(static_cast<const T*>(a.k), a.kb, a.kn, a.kw, hk, dk, a.Hk, max(p.first, k0) - k0, min(p.last, v0) - k0,
        a.per_head ? a.Hq : 1);
  if (!dv || !p.live) return;
  for (int h = max(p.first, v0) - v0; h < p.last - v0; ++h) {
    Pair up{};
    if (hv && there) up = at.load(hv + (((int64_t)p.b * a.Hk + h) * a.N + p.n) * a.D);
    at.store(dv + (p.token * a.Hk + h) * a.D, up);
  }
}

// The weights' gradients: a block for 16 dimensions of each weight row adds up the blocks' sums, in fp64.
template <typename W>
__global__ __launch_bounds__(kSumThr) void k_heads_weights(const float* __restrict__ work, int rows, int D, int split,
                                                           W* __restrict__ dqw, W* __restrict__ dkw) {
  constexpr int kParts = kSumThr / 16;
  __shared__ double sum[kParts][16];
  const int c = threadIdx.x & 15, part = threadIdx.x >> 4, target = blockIdx.x, targets = gridDim.x, d = 16 * blockIdx.y + c;
  double s = 0;
  if (d < D) {
    const float* from = work + (size_t)target * D + d;
#pragma unroll 8
    for (int i = part; i < rows; i += kParts) s += from[(size_t)i * targets * D];
  }
  sum[part][c] = s;
  __syncthreads();
  for (int n = kParts / 2; n > 0; n >>= 1) {
    if (part < n) sum[part][c] += sum[part + n][c];
    __syncthreads();
  }
  W* const dst = target < split ? dqw : dkw;
  if (part == 0 && d < D && dst) put(dst + (size_t)(target < split ? target : target - split) * D + d, (float)sum[0][c]);
}

namespace {
// Rows of 16-byte pieces: lanes move 8 values at once. Value by value the sizes above take 87 and 120 us.
bool wide(const HeadsArgs& a, int size) {
  if ((a.R / 2) % 8 || (a.D - a.R) % 16) return false;
  for (const void* p : {a.q, a.k, a.v, a.qw, a.kw, a.cosine, a.sine})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t s : {a.qb, a.qn, a.kb, a.kn, a.vb, a.vn})
    if (s * size % 16) return false;
  return true;
}
// Blocks for all tokens, and parts of the heads so that there are about `most` blocks: more parts read the tables
// again, fewer leave CUs waiting. At the sizes above the forward takes 17 us with 512 or 2048, 15 with 1024;
// the backward, whose parts leave sums behind, 22 and 3 with 512, 24 and 4 with 1024, 28 and 6 with 2048.
struct Grid {
  int blocks, parts, each;
};
Grid heads_grid(const HeadsArgs& a, int most) {
  const int heads = a.Hq + 2 * a.Hk, blocks = (int)(((int64_t)a.B * a.N + kTokens - 1) / kTokens);
  const int each = (int)std::clamp<int64_t>((int64_t)heads * blocks / most, 1, heads);
  return {blocks, (heads + each - 1) / each, each};
}
constexpr int kForward = 1024, kBackward = 512;
}  // namespace

int heads_blocks(const HeadsArgs& a) {
  const Grid g = heads_grid(a, kBackward);
  return a.per_head ? g.blocks : g.blocks * g.parts;
}

template <typename T>
void launch_heads_forward(const HeadsArgs& a, void* hq, void* hk, void* hv, hipStream_t st, const Timer& timed) {
  const auto kernel = wide(a, sizeof(T)) ? k_heads<T, true> : k_heads<T, false>;
  const Grid g = heads_grid(a, kForward);
  timed("k_heads", st, [&] {
    hipLaunchKernelGGL(kernel, dim3(g.blocks, g.parts), dim3(kThr), 0, st, a, g.each, static_cast<T*>(hq),
                       static_cast<T*>(hk), static_cast<T*>(hv));
  });
}

template <typename T>
void launch_heads_backward(const HeadsArgs& a, const void* hq, const void* hk, const void* hv, void* dq, void* dk,
                           void* dv, void* dqw, void* dkw, float* work, hipStream_t st, const Timer& timed) {
  const auto kernel = wide(a, sizeof(T)) ? k_heads_bwd<T, true> : k_heads_bwd<T, false>;
  const Grid g = heads_grid(a, kBackward);
  timed("k_heads_bwd", st, [&] {
    hipLaunchKernelGGL(kernel, dim3(g.blocks, g.parts), dim3(kThr), 0, st, a, g.each, static_cast<const T*>(hq),
                       static_cast<const T*>(hk), static_cast<const T*>(hv), static_cast<T*>(dq), static_cast<T*>(dk),
                       static_cast<T*>(dv), work);
  });
  if (!work) return;
  const int split = a.per_head ? a.Hq : 1, targets = a.per_head ? a.Hq + a.Hk : 2;
  const dim3 grid(targets, (a.D + 15) / 16), block(kSumThr);
  timed("k_heads_weights", st, [&] {
    if (a.w32)
      hipLaunchKernelGGL(k_heads_weights<float>, grid, block, 0, st, work, heads_blocks(a), a.D, split,
                         static_cast<float*>(dqw), static_cast<float*>(dkw));
    else
      hipLaunchKernelGGL(k_heads_weights<T>, grid, block, 0, st, work, heads_blocks(a), a.D, split, static_cast<T*>(dqw),
                         static_cast<T*>(dkw));
  });
}

#define OAL_HEADS(T)                                                                                                  \
  template void launch_heads_forward<T>(const HeadsArgs&, void*, void*, void*, hipStream_t, const Timer&);            \
  template void launch_heads_backward<T>(const HeadsArgs&, const void*, const void*, const void*, void*, void*,       \
                                         void*, void*, void*, float*, hipStream_t, const Timer&);
OAL_HEADS(float)
OAL_HEADS(uint16_t)
OAL_HEADS(_Float16)
#undef OAL_HEADS

}  // namespace oal
