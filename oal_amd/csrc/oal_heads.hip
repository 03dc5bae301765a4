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
// row, of which each takes 8 pairs of dimensions. A thread stays with one head, so that weights are read once and their
// gradients' sums stay in registers; a block's go to memory, and a second kernel adds those up, in order.
// Arithmetic and sums are in fp32, one rounding to the tensors' type.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "oal_common.hpp"
#include "oal_heads.hpp"
#include "oal_tile.hpp"

namespace oal {

namespace {

constexpr int kThr = 256;
constexpr int kRows = kThr / 4;  // a block's head rows at once
constexpr int kBackBlocks = 512;

__device__ __forceinline__ void store_row8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store_row8(uint16_t* p, const float (&x)[8]) {
  *reinterpret_cast<bf16x8*>(p) = pack8(x);
}
__device__ __forceinline__ void store_row8(_Float16* p, const float (&x)[8]) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  f16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<_Float16>(x[e]);
  *reinterpret_cast<f16x8*>(p) = v;
}

// A lane's 8 pairs (lo, hi) of a row's D values: the first R / 2 pairs are those that the rotation
// turns, (p, p + R / 2), the others two of the rest. With WIDE a lane's lo and hi are 8 values in a row
// each (R / 2 and (D - R) / 2 multiples of 8, rows 16-byte aligned).
template <bool WIDE>
struct Pairs {
  int lo[WIDE ? 1 : 8], hi[WIDE ? 1 : 8];  // -1: none
  bool turned[WIDE ? 1 : 8];
  __device__ __forceinline__ Pairs(int D, int R, int j) {
    const int half = R / 2;
    if constexpr (WIDE) {
      const int p = 8 * j;
      turned[0] = p < half;
      lo[0] = turned[0] ? p : R + 2 * (p - half);
      hi[0] = turned[0] ? p + half : lo[0] + 8;
      if (lo[0] >= D) lo[0] = hi[0] = -1;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = 8 * j + e;
        turned[e] = p < half;
        lo[e] = turned[e] ? p : R + 2 * (p - half);
        hi[e] = turned[e] ? p + half : lo[e] + 1;
        if (lo[e] >= D) lo[e] = -1;
        if (hi[e] >= D) hi[e] = -1;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* p, float (&x)[8], float (&y)[8], float none = 0.f) const {
    if constexpr (WIDE) {
      if (lo[0] >= 0) {
        load_row8(x, p + lo[0]);
        load_row8(y, p + hi[0]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e] = none;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = lo[e] >= 0 ? get(p + lo[e]) : none;
        y[e] = hi[e] >= 0 ? get(p + hi[e]) : none;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* p, const float (&x)[8], const float (&y)[8]) const {
    if constexpr (WIDE) {
      if (lo[0] >= 0) {
        store_row8(p + lo[0], x);
        store_row8(p + hi[0], y);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (lo[e] >= 0) put(p + lo[e], x[e]);
        if (hi[e] >= 0) put(p + hi[e], y[e]);
      }
    }
  }
  // cos and sin of the pairs; those that are not turned by an angle of zero
  template <typename T>
  __device__ __forceinline__ void angles(const T* p, float (&x)[8], float (&y)[8], float none) const {
    if constexpr (WIDE) {
      if (turned[0] && lo[0] >= 0) {
        load_row8(x, p + lo[0]);
        load_row8(y, p + hi[0]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e] = none;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = turned[e] ? get(p + lo[e]) : none;
        y[e] = turned[e] ? get(p + hi[e]) : none;
      }
    }
  }
};

// A sum over the four lanes of a row.
__device__ __forceinline__ float row_sum(float x) {
  x += __shfl_xor(x, 1, 64);
  return x + __shfl_xor(x, 2, 64);
}

// The rows of a block: `tokens` tokens of `heads` heads at once, thread t's the row t / 4. Where there are
// more heads than rows, blockIdx.y takes a part of them.
struct Rows {
  int heads, tokens, first;
  __device__ __forceinline__ explicit Rows(int total) {
    first = blockIdx.y * kRows;
    heads = min(kRows, total - first);
    tokens = kRows / heads;
  }
};

template <typename T>
__device__ __forceinline__ void weights(const HeadsArgs& a, const void* w, int h, const auto& at, float (&x)[8],
                                        float (&y)[8]) {
  const size_t from = a.per_head ? (size_t)h * a.D : 0;
  if (!w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = y[e] = 1.f;
  } else if (a.w32) {
    at.load(static_cast<const float*>(w) + from, x, y);
  } else {
    at.load(static_cast<const T*>(w) + from, x, y);
  }
}
// cos and sin of a position, for the rotation or back. Positions past the tables give NaN.
template <typename T>
__device__ __forceinline__ void table_rows(const HeadsArgs& a, int64_t pos, const auto& at, float (&cl)[8], float (&ch)[8],
                                           float (&sl)[8], float (&sh)[8]) {
  const bool in = pos < a.table;
  const size_t from = in ? (size_t)pos * a.R : 0;
  if (a.t32) {
    at.angles(static_cast<const float*>(a.cosine) + from, cl, ch, 1.f);
    at.angles(static_cast<const float*>(a.sine) + from, sl, sh, 0.f);
  } else {
    at.angles(static_cast<const T*>(a.cosine) + from, cl, ch, 1.f);
    at.angles(static_cast<const T*>(a.sine) + from, sl, sh, 0.f);
  }
  if (!in) {
#pragma unroll
    for (int e = 0; e < 8; ++e) cl[e] = ch[e] = __builtin_nanf("");
  }
}

}  // namespace

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThr) void k_heads(HeadsArgs a, T* __restrict__ hq, T* __restrict__ hk, T* __restrict__ hv) {
  const Rows rows(a.Hq + 2 * a.Hk);
  const int slot = threadIdx.x >> 2, hh = rows.first + slot % rows.heads;
  if (slot >= rows.tokens * rows.heads) return;
  const Pairs<WIDE> at(a.D, a.R, threadIdx.x & 3);
  const bool is_q = hh < a.Hq, is_v = hh >= a.Hq + a.Hk;
  const int h = is_q ? hh : is_v ? hh - a.Hq - a.Hk : hh - a.Hq, H = is_q ? a.Hq : a.Hk;
  const T* src = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) + (size_t)h * a.D;
  const int64_t sb = is_q ? a.qb : is_v ? a.vb : a.kb, sn = is_q ? a.qn : is_v ? a.vn : a.kn;
  T* const dst = is_q ? hq : is_v ? hv : hk;
  float wl[8], wh[8];
  if (!is_v) weights<T>(a, is_q ? a.qw : a.kw, h, at, wl, wh);
  const int64_t total = (int64_t)a.B * a.N;
  for (int64_t i = (int64_t)blockIdx.x * rows.tokens + slot / rows.heads; i < total; i += (int64_t)gridDim.x * rows.tokens) {
    const int64_t b = i / a.N, n = i % a.N;
    const int64_t pos = a.position ? a.position[i] : n;
    float lo[8], hi[8];
    at.load(src + b * sb + n * sn, lo, hi);
    if (!is_v) {
      float cl[8], ch[8], sl[8], sh[8], sum = 0.f;
      table_rows<T>(a, pos < 0 ? 0 : pos, at, cl, ch, sl, sh);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += lo[e] * lo[e] + hi[e] * hi[e];
      const float r = 1.f / sqrtf(row_sum(sum) / a.D + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = lo[e] * r * wl[e], y = hi[e] * r * wh[e];
        lo[e] = x * cl[e] - y * sl[e];
        hi[e] = y * ch[e] + x * sh[e];
      }
    }
    if (pos < 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.f;
    }
    at.store(dst + ((b * H + h) * a.N + n) * a.D, lo, hi);
  }
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThr) void k_heads_bwd(HeadsArgs a, const T* __restrict__ hq, const T* __restrict__ hk,
                                                    const T* __restrict__ hv, T* __restrict__ dq, T* __restrict__ dk,
                                                    T* __restrict__ dv, float* __restrict__ work) {
  __shared__ alignas(16) float sums[kRows][68];
  const Rows rows(a.Hq + 2 * a.Hk);
  const int slot = threadIdx.x >> 2, hh = rows.first + slot % rows.heads;
  const bool live = slot < rows.tokens * rows.heads;
  const Pairs<WIDE> at(a.D, a.R, threadIdx.x & 3);
  const bool is_q = hh < a.Hq, is_v = hh >= a.Hq + a.Hk;
  const int h = is_q ? hh : is_v ? hh - a.Hq - a.Hk : hh - a.Hq, H = is_q ? a.Hq : a.Hk;
  const T* up = is_q ? hq : is_v ? hv : hk;
  T* const dst = is_q ? dq : is_v ? dv : dk;
  const T* src = static_cast<const T*>(is_q ? a.q : a.k) + (size_t)h * a.D;
  const int64_t sb = is_q ? a.qb : a.kb, sn = is_q ? a.qn : a.kn;
  float wl[8], wh[8], gl[8] = {}, gh[8] = {};
  if (!is_v) weights<T>(a, is_q ? a.qw : a.kw, h, at, wl, wh);
  const int64_t total = live && dst ? (int64_t)a.B * a.N : 0;
  for (int64_t i = (int64_t)blockIdx.x * rows.tokens + slot / rows.heads; i < total; i += (int64_t)gridDim.x * rows.tokens) {
    const int64_t b = i / a.N, n = i % a.N;
    const int64_t pos = a.position ? a.position[i] : n;
    float lo[8] = {}, hi[8] = {};
    if (up && pos >= 0) at.load(up + ((b * H + h) * a.N + n) * a.D, lo, hi);
    if (!is_v) {
      float cl[8], ch[8], sl[8], sh[8], xl[8], xh[8], sum = 0.f, dot = 0.f;
      at.load(src + b * sb + n * sn, xl, xh);
      table_rows<T>(a, pos < 0 ? 0 : pos, at, cl, ch, sl, sh);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = lo[e], y = hi[e];
        lo[e] = x * cl[e] + y * sh[e];
        hi[e] = y * ch[e] - x * sl[e];
        sum += xl[e] * xl[e] + xh[e] * xh[e];
      }
      const float r = 1.f / sqrtf(row_sum(sum) / a.D + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xl[e] *= r, xh[e] *= r;
        if (pos >= 0) gl[e] += xl[e] * lo[e], gh[e] += xh[e] * hi[e];
        lo[e] *= wl[e], hi[e] *= wh[e];
        dot += xl[e] * lo[e] + xh[e] * hi[e];
      }
      dot = row_sum(dot) / a.D;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = pos < 0 ? 0.f : r * (lo[e] - xl[e] * dot);
        hi[e] = pos < 0 ? 0.f : r * (hi[e] - xh[e] * dot);
      }
    }
    at.store(dst + ((int64_t)i * H + h) * a.D, lo, hi);
  }
  if (!work) return;
  // the block's sums of each weight's gradient, rows in order
  if (live && !is_v) at.store(sums[slot], gl, gh);
  __syncthreads();
  const int targets = a.per_head ? a.Hq + a.Hk : 2;
  for (int x = threadIdx.x; x < targets * a.D; x += kThr) {
    const int target = x / a.D, d = x % a.D;
    float s = 0.f;
    for (int i = 0; i < rows.tokens * rows.heads; ++i) {
      const int head = rows.first + i % rows.heads;
      if (head >= a.Hq + a.Hk) continue;
      if ((a.per_head ? head : head >= a.Hq) == target) s += sums[i][d];
    }
    work[((size_t)(blockIdx.y * gridDim.x + blockIdx.x) * targets + target) * a.D + d] = s;
  }
}

// The weights' gradients: a block for each weight row adds up the blocks' sums, in fp64.
template <typename W>
__global__ __launch_bounds__(kThr) void k_heads_weights(const float* __restrict__ work, int blocks, int D, int split,
                                                        W* __restrict__ dqw, W* __restrict__ dkw) {
  __shared__ double sum[kThr / 64][64];
  const int d = threadIdx.x & 63, part = threadIdx.x >> 6, target = blockIdx.x, targets = gridDim.x;
  double s = 0;
  if (d < D)
    for (int i = part; i < blocks; i += kThr / 64) s += work[((size_t)i * targets + target) * D + d];
  sum[part][d] = s;
  __syncthreads();
  if (part || d >= D) return;
  W* const dst = target < split ? dqw : dkw;
  if (dst) put(dst + (size_t)(target < split ? target : target - split) * D + d, (float)((sum[0][d] + sum[1][d]) + (sum[2][d] + sum[3][d])));
}

namespace {
// Rows of 16-byte pieces: lanes move 8 values at once.
bool wide(const HeadsArgs& a, int size) {
  if ((a.R / 2) % 8 || (a.D - a.R) % 16) return false;
  for (const void* p : {a.q, a.k, a.v, a.qw, a.kw, a.cosine, a.sine})
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t s : {a.qb, a.qn, a.kb, a.kn, a.vb, a.vn})
    if (s * size % 16) return false;
  return true;
}
dim3 heads_grid(const HeadsArgs& a, int most) {
  const int heads = a.Hq + 2 * a.Hk, parts = (heads + kRows - 1) / kRows, tokens = kRows / std::min(heads, kRows);
  const int64_t blocks = ((int64_t)a.B * a.N + tokens - 1) / tokens;
  return dim3((unsigned)std::min<int64_t>(blocks, most), parts);
}
}  // namespace

int heads_blocks(const HeadsArgs& a) {
  const dim3 g = heads_grid(a, kBackBlocks);
  return g.x * g.y;
}

template <typename T>
void launch_heads_forward(const HeadsArgs& a, void* hq, void* hk, void* hv, hipStream_t st, const Timer& timed) {
  const auto kernel = wide(a, sizeof(T)) ? k_heads<T, true> : k_heads<T, false>;
  timed("k_heads", st, [&] {
    hipLaunchKernelGGL(kernel, heads_grid(a, 4096), dim3(kThr), 0, st, a, static_cast<T*>(hq), static_cast<T*>(hk),
                       static_cast<T*>(hv));
  });
}

template <typename T>
void launch_heads_backward(const HeadsArgs& a, const void* hq, const void* hk, const void* hv, void* dq, void* dk,
                           void* dv, void* dqw, void* dkw, float* work, hipStream_t st, const Timer& timed) {
  const auto kernel = wide(a, sizeof(T)) ? k_heads_bwd<T, true> : k_heads_bwd<T, false>;
  const dim3 grid = heads_grid(a, kBackBlocks);
  timed("k_heads_bwd", st, [&] {
    hipLaunchKernelGGL(kernel, grid, dim3(kThr), 0, st, a, static_cast<const T*>(hq), static_cast<const T*>(hk),
                       static_cast<const T*>(hv), static_cast<T*>(dq), static_cast<T*>(dk), static_cast<T*>(dv), work);
  });
  if (!work) return;
  const int split = a.per_head ? a.Hq : 1, targets = a.per_head ? a.Hq + a.Hk : 2;
  timed("k_heads_weights", st, [&] {
    if (a.w32)
      hipLaunchKernelGGL(k_heads_weights<float>, dim3(targets), dim3(kThr), 0, st, work, (int)(grid.x * grid.y), a.D,
                         split, static_cast<float*>(dqw), static_cast<float*>(dkw));
    else
      hipLaunchKernelGGL(k_heads_weights<T>, dim3(targets), dim3(kThr), 0, st, work, (int)(grid.x * grid.y), a.D, split,
                         static_cast<T*>(dqw), static_cast<T*>(dkw));
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
