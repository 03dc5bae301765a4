// Log probabilities of given tokens for gfx950, with the entropy of their distributions and the
// most likely alternatives, in one pass over the logits; and the gradient in another.
//
//   m = max_v x_v,  s = sum_v e^(x_v - m),  t = sum_v e^(x_v - m) (x_v - m)
//   log p_v = x_v - m - log s,  H = -sum_v p_v log p_v = log s - t / s
//   dx_v = dlog (1 if v is the token - p_v) - dH p_v (log p_v + H)
//
// Bound by memory: a row is read once, 16 bytes per lane, with running maxima and sums per lane that
// are joined at the end. Rows are cut into parts where there are fewer than fill the GPU, and a
// second kernel joins those. All of it is in fp32: differences to the maximum are exact for 16-bit logits.
//
// The alternatives: a wave keeps the highest 64 of its values so far in order, one per lane, and
// looks at a value only if it comes before the last that counts; of equal values the first. A row of random
// order changes that list some K log(V / K) times.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "oal_common.hpp"
#include "oal_scores.hpp"
#include "oal_tile.hpp"

namespace oal {

namespace {

constexpr int kThr = 256;
constexpr int kWaves = kThr / 64;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A row's running sums.
struct Sums {
  float m, s, t;
};
constexpr Sums kNothing = {-INFINITY, 0.f, 0.f};
// What sums over values with maximum m become with the maximum `to`, which is not lower.
__device__ __forceinline__ void move_to(Sums& x, float to) {
  if (x.m == to || x.s == 0.f) {
    x.m = to;
    return;
  }
  const float d = x.m - to, c = exp_of(d);
  // what vanishes leaves nothing, and not zero times infinity
  x.t = c > 0.f ? (x.t + x.s * d) * c : 0.f;
  x.s *= c;
  x.m = to;
}
__device__ __forceinline__ void join(Sums& a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  move_to(a, m);
  move_to(b, m);
  a.s += b.s;
  a.t += b.t;
}

// Adds N values.
template <int N, bool ENTROPY>
__device__ __forceinline__ void add(Sums& a, const float (&x)[N]) {
  float most = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
  if (most > a.m) move_to(a, most);
  const float m = a.m == -INFINITY ? 0.f : a.m;  // -inf values weigh nothing
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float z = x[e] - m, y = exp_of(z);
    a.s += y;
    // 0 times -inf is no share
    if (ENTROPY) a.t = fmaf(y, fmaxf(z, -1e30f), a.t);
  }
}

// A wave's highest values in order, one per lane. Empty places are below all values, -inf too.
struct Best {
  float x = -INFINITY;
  uint32_t at = 0xffffffffu;
  // the last that counts, the same in all lanes
  float last = -INFINITY;
  uint32_t last_at = 0xffffffffu;
};
__device__ __forceinline__ bool before(float x, uint32_t i, float y, uint32_t j) { return x > y || (x == y && i < j); }
__device__ __forceinline__ float lane_f(float x, int l) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
}
__device__ __forceinline__ uint32_t lane_u(uint32_t x, int l) { return __builtin_amdgcn_readlane(x, l); }

// All lanes: value x of place i, which is the same in all, takes its place.
__device__ __forceinline__ void insert(Best& b, float x, uint32_t i, int top, int lane) {
  const bool behind = before(x, i, b.x, b.at);
  const float px = __shfl_up(b.x, 1, 64);
  const uint32_t pi = __shfl_up(b.at, 1, 64);
  const bool prev = lane > 0 && before(x, i, px, pi);
  if (behind) {
    b.x = prev ? px : x;
    b.at = prev ? pi : i;
  }
  b.last = lane_f(b.x, top - 1);
  b.last_at = lane_u(b.at, top - 1);
}
// Each lane's N values of places i, i + 1, ...
template <int N>
__device__ __forceinline__ void offer(Best& b, const float (&x)[N], uint32_t i, bool in, int top, int lane) {
  float most = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
  if (!__ballot(in && before(most, i, b.last, b.last_at))) return;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    uint64_t who = __ballot(in && before(x[e], i + e, b.last, b.last_at));
    while (who) {
      const int l = __ffsll((unsigned long long)who) - 1;
      insert(b, lane_f(x[e], l), lane_u(i + e, l), top, lane);
      who &= who - 1;
      who &= __ballot(in && before(x[e], i + e, b.last, b.last_at));
    }
  }
}

// What a part of a row leaves: its sums, then the values of its best and their places.
struct Part {
  float m, s, t, unused;
};

template <typename T>
constexpr int kPiece = 16 / sizeof(T);

template <typename T>
__device__ __forceinline__ void load_piece(float (&x)[kPiece<T>], const T* p) {
  if constexpr (kPiece<T> == 8) {
    load_row8(x, p);
  } else {
    const f32x4 v = load4(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e];
  }
}

// Where part p of `parts` of a row begins, in pieces from the row's first 16-byte boundary.
__device__ __forceinline__ int64_t part_begin(int64_t pieces, int p, int parts) { return pieces * p / parts; }

}  // namespace

// Merges the waves' lists of `count` places each in LDS: every entry counts those that come before it, and its
// count is its place.
__device__ __forceinline__ void place_best(const float* x, const uint32_t* at, int lists, int top, const auto& put_at) {
  for (int i = threadIdx.x; i < lists * top; i += kThr) {
    const float v = x[i];
    const uint32_t j = at[i];
    int rank = 0;
    for (int n = 0; n < lists * top; ++n) rank += before(x[n], at[n], v, j) || (at[n] == j && x[n] == v && n < i);
    if (rank < top) put_at(rank, v, j);
  }
}

// One part of one row. With parts == 1 it writes the row's results.
template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kThr) void k_scores(ScoreArgs a, ScoreOut out, int parts, Part* __restrict__ sums,
                                                 float* __restrict__ best, uint32_t* __restrict__ best_at) {
  constexpr int P = kPiece<T>;
  __shared__ Sums shared[kWaves];
  __shared__ float bx[TOP ? kWaves * kMostTop : 1];
  __shared__ uint32_t bi[TOP ? kWaves * kMostTop : 1];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t);
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const T* x = static_cast<const T*>(a.logits) + row / a.N * a.b + row % a.N * a.n;
  // values before the first boundary, whole pieces, values behind the last
  const int lead = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), a.V);
  const int64_t pieces = (a.V - lead) / P;
  const int tail = lead + (int)pieces * P;
  const int64_t first = part_begin(pieces, part, parts), end = part_begin(pieces, part + 1, parts);
  Sums mine = kNothing;
  Best b;
  auto take = [&](auto& v, uint32_t i, bool in) {
    constexpr int N = sizeof(v) / sizeof(v[0]);
    if (in) add<N, ENTROPY>(mine, v);
    if constexpr (TOP) offer<N>(b, v, i, in, a.top, lane);
  };
  if (part == 0 && w == 0) {
    float v[1] = {t < lead ? get(x + t) : -INFINITY};
    take(v, t, t < lead);
  }
  // whole waves: a list belongs to all lanes
  for (int64_t i = first; i < end; i += kThr) {
    const int64_t p = i + t;
    const bool in = p < end;
    float v[P];
    load_piece<T>(v, x + lead + (in ? p : first) * P);
    take(v, (uint32_t)(lead + p * P), in);
  }
  if (part == parts - 1 && w == kWaves - 1) {
    float v[1] = {tail + lane < a.V ? get(x + tail + lane) : -INFINITY};
    take(v, tail + lane, tail + lane < a.V);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const Sums other = {__shfl_xor(mine.m, off, 64), __shfl_xor(mine.s, off, 64), __shfl_xor(mine.t, off, 64)};
    join(mine, other);
  }
  if (lane == 0) shared[w] = mine;
  if constexpr (TOP) {
    if (lane < a.top) bx[w * a.top + lane] = b.x, bi[w * a.top + lane] = b.at;
  }
  __syncthreads();
  mine = shared[0];
#pragma unroll
  for (int n = 1; n < kWaves; ++n) join(mine, shared[n]);
  if (parts > 1) {
    if (t == 0) sums[blockIdx.x] = {mine.m, mine.s, mine.t, 0.f};
    if constexpr (TOP) {
      place_best(bx, bi, kWaves, a.top, [&](int rank, float v, uint32_t j) {
        best[(size_t)blockIdx.x * a.top + rank] = v;
        best_at[(size_t)blockIdx.x * a.top + rank] = j;
      });
    }
    return;
  }
  const float log = logf(mine.s);
  if (t == 0) {
    const int64_t token = a.tokens[row];
    out.logp[row] = token < 0 ? 0.f : token < a.V ? get(x + token) - mine.m - log : __builtin_nanf("");
    if (ENTROPY) out.entropy[row] = log - mine.t / mine.s;
    if (out.saved) out.saved[2 * row] = mine.m, out.saved[2 * row + 1] = mine.s;
  }
  if constexpr (TOP) {
    place_best(bx, bi, kWaves, a.top, [&](int rank, float v, uint32_t j) {
      out.top[row * a.top + rank] = v - mine.m - log;
      out.place[row * a.top + rank] = j == 0xffffffffu ? -1 : (int64_t)j;
    });
  }
}

// The parts of one row, joined.
template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kThr) void k_scores_join(ScoreArgs a, ScoreOut out, int parts, const Part* __restrict__ sums,
                                                      const float* __restrict__ best,
                                                      const uint32_t* __restrict__ best_at) {
  extern __shared__ char room[];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  Sums mine = kNothing;
  for (int p = 0; p < parts; ++p) {
    const Part x = sums[row * parts + p];
    join(mine, {x.m, x.s, x.t});
  }
  const float log = logf(mine.s);
  if (t == 0) {
    const T* x = static_cast<const T*>(a.logits) + row / a.N * a.b + row % a.N * a.n;
    const int64_t token = a.tokens[row];
    out.logp[row] = token < 0 ? 0.f : token < a.V ? get(x + token) - mine.m - log : __builtin_nanf("");
    if (ENTROPY) out.entropy[row] = log - mine.t / mine.s;
    if (out.saved) out.saved[2 * row] = mine.m, out.saved[2 * row + 1] = mine.s;
  }
  if constexpr (TOP) {
    const int count = parts * a.top;
    float* bx = reinterpret_cast<float*>(room);
    uint32_t* bi = reinterpret_cast<uint32_t*>(bx + count);
    for (int i = t; i < count; i += kThr) bx[i] = best[row * count + i], bi[i] = best_at[row * count + i];
    __syncthreads();
    place_best(bx, bi, parts, a.top, [&](int rank, float v, uint32_t j) {
      out.top[row * a.top + rank] = v - mine.m - log;
      out.place[row * a.top + rank] = j == 0xffffffffu ? -1 : (int64_t)j;
    });
  }
}

// The gradient of one part of one row.
template <typename T>
__global__ __launch_bounds__(kThr) void k_scores_bwd(ScoreArgs a, int parts, const float* __restrict__ saved,
                                                     const float* __restrict__ entropy, const float* __restrict__ dlog,
                                                     const float* __restrict__ dentropy, T* __restrict__ dlogits) {
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const T* x = static_cast<const T*>(a.logits) + row / a.N * a.b + row % a.N * a.n;
  T* dx = dlogits + row * a.V;
  const int64_t token = a.tokens[row];
  const float m = saved[2 * row], s = saved[2 * row + 1], log = logf(s), inv = 1.f / s;
  float dl = dlog && token >= 0 ? dlog[row] : 0.f;
  if (token >= a.V) dl *= __builtin_nanf("");
  const float dh = dentropy ? dentropy[row] : 0.f, base = dentropy ? entropy[row] - log : 0.f;
  const int from = (int)((int64_t)a.V * part / parts), to = (int)((int64_t)a.V * (part + 1) / parts);
  for (int v = from + t; v < to; v += kThr) {
    const float z = get(x + v) - m, p = exp_of(z) * inv;
    put(dx + v, (v == token ? dl : 0.f) - p * (dl + dh * (fmaxf(z, -1e30f) + base)));
  }
}

namespace {
int score_parts(const ScoreArgs& a) {
  const int64_t rows = (int64_t)a.B * a.N;
  // a part has two turns of the block's 16-byte pieces or more
  const int64_t most = std::max(1, a.V / (kThr * 16));
  return (int)std::clamp<int64_t>((1024 + rows - 1) / rows, 1, std::min<int64_t>(most, 64));
}
}  // namespace

size_t score_work_bytes(const ScoreArgs& a) {
  const int parts = score_parts(a);
  if (parts == 1) return 0;
  return (size_t)a.B * a.N * parts * (sizeof(Part) + 8 * a.top);
}

template <typename T>
void launch_scores(const ScoreArgs& a, const ScoreOut& out, void* work, hipStream_t st, const Timer& timed) {
  const int parts = score_parts(a);
  const int64_t rows = (int64_t)a.B * a.N;
  Part* sums = static_cast<Part*>(work);
  float* best = reinterpret_cast<float*>(sums + rows * parts);
  uint32_t* best_at = reinterpret_cast<uint32_t*>(best + rows * parts * a.top);
  auto launch = [&](auto kernel, auto second) {
    timed("k_scores", st, [&] {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * parts)), dim3(kThr), 0, st, a, out, parts, sums, best, best_at);
    });
    if (parts > 1)
      timed("k_scores_join", st, [&] {
        hipLaunchKernelGGL(second, dim3((unsigned)rows), dim3(kThr), (size_t)8 * parts * a.top, st, a, out, parts, sums,
                           best, best_at);
      });
  };
  if (a.top && a.entropy)
    launch(k_scores<T, true, true>, k_scores_join<T, true, true>);
  else if (a.top)
    launch(k_scores<T, false, true>, k_scores_join<T, false, true>);
  else if (a.entropy)
    launch(k_scores<T, true, false>, k_scores_join<T, true, false>);
  else
    launch(k_scores<T, false, false>, k_scores_join<T, false, false>);
}

template <typename T>
void launch_scores_backward(const ScoreArgs& a, const float* saved, const float* entropy, const float* dlog,
                            const float* dentropy, void* dlogits, hipStream_t st, const Timer& timed) {
  const int parts = score_parts(a);
  timed("k_scores_bwd", st, [&] {
    hipLaunchKernelGGL(k_scores_bwd<T>, dim3((unsigned)((int64_t)a.B * a.N * parts)), dim3(kThr), 0, st, a, parts, saved,
                       entropy, dlog, dentropy, static_cast<T*>(dlogits));
  });
}

#define OAL_SCORES(T)                                                                                               \
  template void launch_scores<T>(const ScoreArgs&, const ScoreOut&, void*, hipStream_t, const Timer&);              \
  template void launch_scores_backward<T>(const ScoreArgs&, const float*, const float*, const float*, const float*, \
                                          void*, hipStream_t, const Timer&);
OAL_SCORES(float)
OAL_SCORES(uint16_t)
OAL_SCORES(_Float16)
#undef OAL_SCORES

}  // namespace oal
