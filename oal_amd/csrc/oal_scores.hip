// Log probabilities of given tokens for gfx950, with the entropy of their distributions and the
// most likely alternatives, in one pass over the logits; and the gradient in another.
//
//   m = max_v x_v,  s = sum_v e^(x_v - m),  t = sum_v e^(x_v - m) (x_v - m)
//   log p_v = x_v - m - log s,  H = -sum_v p_v log p_v = log s - t / s
//   dx_v = dlog (1 if v is the token - p_v) - dH p_v (log p_v + H)
//
// Bound by memory: a row is read once, 16 bytes per lane, with a running maximum per wave and sums per lane that
// are joined at the end. Rows are cut into parts where there are fewer than fill the GPU, and a
// second kernel joins those. A value's difference z to the maximum is one rounding in fp32, and its exponential is off by
// that of z log2 e, up to 2^-24 |z|, and one more; sums are in fp64.
//
// 2 x 1000 rows of 151936 bf16 logits with the entropy: forward 150 us (608 MB, 4.1 TB/s), gradient 229 us (1216 MB,
// 5.3 TB/s). 4096 rows with five alternatives: 266 us (1245 MB, 4.7 TB/s). Beside the loads a value costs about ten
// instructions, an exponential of four times the price among them. One row with 20 alternatives: 13 us in 49 parts, whose loads
// are waited for one by one (score_parts) while the lists begin, and 7 to join them;
// 48 rows of 32003 fp32 logits in 10 parts each: 16 and 5.
//
// The alternatives: a wave keeps the highest 64 of its values so far in order, one per lane, and
// looks at a value only if it comes before the last that counts; of equal values the first. A row of random
// order changes that list some K log(V / K) times. Where many lanes have such a value they are
// sorted and merged with the list at once, as at the beginning; else they move up the list one by one.

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
// A logarithm whose exponential is zero: lower ones, -inf among them, are this where they are multiplied with it.
constexpr float kGone = -200.f;

// A row's running sums, in 64 bits: of a row with nearly all weight in one place s is 1 and what is asked for. In 32 bits
// the other values of that place's lane were lost, 2e-3 of a log probability of -3e-4 and 1e-4 of the row's entropy.
struct Sums {
  float m;
  double s, t;
};
constexpr Sums kNothing = {-INFINITY, 0, 0};
// What sums over values with maximum m become with the maximum `to`, which is not lower.
__device__ __forceinline__ void move_to(Sums& x, float to) {
  if (x.m == to || x.s == 0) {
    x.m = to;
    return;
  }
  const float d = x.m - to, c = exp_of(d);
  // what vanishes leaves nothing, and not zero times infinity
  x.t = c > 0.f ? (x.t + x.s * d) * c : 0;
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

template <int N>
__device__ __forceinline__ float most_of(const float (&x)[N]) {
  float most = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
  return most;
}
// A turn's values, before they go to the sums: 4096 rows take 268 us, with each piece's going there by itself 275, with
// sums in 32 bits 260.
struct Few {
  float s = 0.f, t = 0.f;
  __device__ __forceinline__ void to(Sums& a) {
    a.s += s;
    a.t += t;
    s = t = 0.f;
  }
};
// Adds each lane's N values, the highest of them `most`; all lanes. They are taken relative to the wave's maximum so far,
// of which the exponential is one. It seldom moves; the values that come with a new one are added one by one in 64 bits.
template <int N, bool ENTROPY>
__device__ __forceinline__ void add(Sums& a, Few& few, const float (&x)[N], float most) {
  const bool moves = __any(most > a.m);
  if (moves) {
    few.to(a);
    float to = fmaxf(most, a.m);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) to = fmaxf(to, __shfl_xor(to, off, 64));
    move_to(a, __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(to))));
  }
  const float m = a.m == -INFINITY ? 0.f : a.m;  // -inf values weigh nothing
  auto each = [&](auto& s, auto& t) {
    typedef std::remove_reference_t<decltype(s)> S;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float z = x[e] - m, y = exp_of(z);
      s += y;
      if (ENTROPY) t = fma((S)y, (S)fmaxf(z, kGone), t);
    }
  };
  if (moves)
    each(a.s, a.t);
  else
    each(few.s, few.t);
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
__device__ __forceinline__ void insert(Best& b, float x, uint32_t i) {
  // from the lane before (wave_shr:1); lane 0 keeps what it had, which is behind nothing
  const float px = __int_as_float(__builtin_amdgcn_update_dpp(0x7f800000, __float_as_int(b.x), 0x138, 0xf, 0xf, false));
  const uint32_t pi = __builtin_amdgcn_update_dpp(0, b.at, 0x138, 0xf, 0xf, false);
  const bool behind = before(x, i, b.x, b.at), prev = before(x, i, px, pi);
  b.x = prev ? px : behind ? x : b.x;
  b.at = prev ? pi : behind ? i : b.at;
}

// The value of the lane `WITH` away (lane ^ WITH), by lane moves alone: through LDS a step of the network below would
// wait for its answer.
template <int WITH>
__device__ __forceinline__ uint32_t partner(uint32_t x, int lane) {
  auto move = [](uint32_t v, auto how) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(how)::value, 0xf, 0xf, true);
  };
  if constexpr (WITH == 1)
    return move(x, std::integral_constant<int, 0xb1>());  // quad_perm:[1,0,3,2]
  else if constexpr (WITH == 2)
    return move(x, std::integral_constant<int, 0x4e>());  // quad_perm:[2,3,0,1]
  else if constexpr (WITH == 4)  // lane ^ 7 (row_half_mirror), then ^ 3 (quad_perm:[3,2,1,0])
    return move(move(x, std::integral_constant<int, 0x141>()), std::integral_constant<int, 0x1b>());
  else if constexpr (WITH == 8)
    return move(x, std::integral_constant<int, 0x128>());  // row_ror:8
  else if constexpr (WITH == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
// One step of a sorting network: the lane keeps the earlier or the later of its own and its partner's.
template <int WITH>
__device__ __forceinline__ void exchange(float& x, uint32_t& i, bool earlier, int lane) {
  const float y = __uint_as_float(partner<WITH>(__float_as_uint(x), lane));
  const uint32_t j = partner<WITH>(i, lane);
  if (before(y, j, x, i) == earlier) x = y, i = j;
}
// Steps of WITH, WITH / 2, ... 1 lanes, towards earlier in the lower lanes where `down`.
template <int WITH>
__device__ __forceinline__ void settle(float& x, uint32_t& i, bool down, int lane) {
  exchange<WITH>(x, i, ((lane & WITH) == 0) == down, lane);
  if constexpr (WITH > 1) settle<WITH / 2>(x, i, down, lane);
}
// All lanes: values x of places i (or none: -inf, 0xffffffff), sorted from the last to the first, into the list. They
// and the list are a sequence that falls and rises, whose 64 highest six steps put in order. Values with equal places
// are empty ones and change nothing, whichever is taken.
__device__ __forceinline__ void merge_sorted(Best& b, float x, uint32_t i, int lane) {
  if (before(x, i, b.x, b.at)) b.x = x, b.at = i;
  settle<32>(b.x, b.at, true, lane);
}
// The same, in any order.
__device__ __forceinline__ void merge(Best& b, float x, uint32_t i, int lane) {
  settle<1>(x, i, lane & 2, lane);
  settle<2>(x, i, lane & 4, lane);
  settle<4>(x, i, lane & 8, lane);
  settle<8>(x, i, lane & 16, lane);
  settle<16>(x, i, lane & 32, lane);
  settle<32>(x, i, false, lane);
  merge_sorted(b, x, i, lane);
}

// Lanes with a value to merge from which that is faster than one by one: 4096 rows with five alternatives took 306 us with
// 3, 294 with 6, 293 with 12 and 292 with 20 before the other steps here.
constexpr int kMerge = 12;
// Waves that join the parts' lists, 4 to a wave at most: 6 us for one row; four waves, sorting them anew, took 17.
constexpr int kJoin = 16;

// Each lane's N values of places i, i + 1, ... (`in`: it has some); `most` is their maximum. Another wave of the
// row has as many values as count that are not below `limit`.
template <int N>
__device__ __forceinline__ void offer(Best& b, float (&x)[N], float most, uint32_t i, bool in, float limit, int top,
                                      int lane) {
  if (!__ballot(in && most >= limit && before(most, i, b.last, b.last_at))) return;
  // one value of each lane at a time, its highest; what has been looked at becomes NaN, which comes before nothing
  for (;;) {
    float v = -INFINITY;
    uint32_t e = N;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (x[n] > v || (x[n] == v && e == N)) v = x[n], e = n;
    const bool take = in && e < N && v >= limit && before(v, i + e, b.last, b.last_at);
    uint64_t who = __ballot(take);
    if (!who) return;
    if (__popcll(who) >= kMerge) {
      merge(b, take ? v : -INFINITY, take ? i + e : 0xffffffffu, lane);
    } else {
      for (; who; who &= who - 1) {
        const int l = __ffsll((unsigned long long)who) - 1;
        insert(b, lane_f(v, l), lane_u(i + e, l));
      }
    }
    b.last = lane_f(b.x, top - 1);
    b.last_at = lane_u(b.at, top - 1);
    for (int n = 0; n < N; ++n)
      if (take && n == (int)e) x[n] = __builtin_nanf("");
  }
}

// What a part of a row leaves: its sums, then the values of its best and their places.
struct Part {
  double s, t;
  float m;
};

template <typename T>
constexpr int kPiece = 16 / sizeof(T);
// Pieces of a lane in flight at once, in the forward with as many of the next turn: with 2, 3 and 4 the 4096 rows take 262,
// 266 and 260 us, 2 x 1000 rows forward 153, 152 and 152, back 230, 227 and 226, 48 short rows 20, 21 and 24. Without the
// next turn on its way the forward takes 267 and 156.
constexpr int kTurn = 3;

// 16 bytes of a row, at any address of its type: rows of an odd vocabulary begin where they may.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Raw {
  uint32_t w[4];
};
template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T* p) {
  return *reinterpret_cast<const Raw<T>*>(p);
}
__device__ __forceinline__ void values(float (&x)[4], const Raw<float>& r) {
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(r.w[e]);
}
__device__ __forceinline__ void values(float (&x)[8], const Raw<uint16_t>& r) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(r.w[e] << 16);
    x[2 * e + 1] = __uint_as_float(r.w[e] & 0xffff0000u);
  }
}
__device__ __forceinline__ void values(float (&x)[8], const Raw<_Float16>& r) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f16x2 v = __builtin_bit_cast(f16x2, (uint32_t)r.w[e]);
    x[2 * e] = static_cast<float>(v[0]);
    x[2 * e + 1] = static_cast<float>(v[1]);
  }
}
__device__ __forceinline__ void store_raw(float* p, const float (&x)[4]) {
  Raw<float> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.w[e] = __float_as_uint(x[e]);
  *reinterpret_cast<Raw<float>*>(p) = r;
}
__device__ __forceinline__ void store_raw(uint16_t* p, const float (&x)[8]) {
  Raw<uint16_t> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
  *reinterpret_cast<Raw<uint16_t>*>(p) = r;
}
__device__ __forceinline__ void store_raw(_Float16* p, const float (&x)[8]) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  Raw<_Float16> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f16x2 v = {static_cast<_Float16>(x[2 * e]), static_cast<_Float16>(x[2 * e + 1])};
    r.w[e] = __builtin_bit_cast(uint32_t, v);
  }
  *reinterpret_cast<Raw<_Float16>*>(p) = r;
}

template <typename T>
__device__ __forceinline__ const T* row_at(const ScoreArgs& a, int64_t row) {
  return static_cast<const T*>(a.logits) + row / a.N * a.b + row % a.N * a.n;
}

// The lists of a block's W waves become the first wave's, half of them into the other half at a time.
template <int W>
struct Lists {
  float x[W][64];
  uint32_t at[W][64];
};
template <int W, int HALF = W / 2>
__device__ __forceinline__ void join_lists(Best& b, Lists<W>& lists, int w, int lane) {
  if (w >= HALF && w < 2 * HALF) lists.x[w][lane] = b.x, lists.at[w][lane] = b.at;
  __syncthreads();
  if (w < HALF) merge_sorted(b, lists.x[w + HALF][63 - lane], lists.at[w + HALF][63 - lane], lane);
  if constexpr (HALF > 1) join_lists<W, HALF / 2>(b, lists, w, lane);
}

// A row's results from its sums and the first wave's list.
template <typename T, bool ENTROPY, bool TOP>
__device__ __forceinline__ void finish(const ScoreArgs& a, const ScoreOut& out, int64_t row, const Sums& sum,
                                       const Best& b) {
  const int t = threadIdx.x;
  const double lse = sum.m + log(sum.s);
  if (t == 0) {
    const int64_t token = a.tokens[row];
    out.logp[row] = token < 0        ? 0.f
                    : token < a.V ? (float)(get(row_at<T>(a, row) + token) - lse)
                                  : __builtin_nanf("");
    if (ENTROPY) out.entropy[row] = (float)(log(sum.s) - sum.t / sum.s);
    if (out.saved) out.saved[2 * row] = sum.m, out.saved[2 * row + 1] = (float)sum.s;
  }
  if (TOP && t < a.top) {
    out.top[row * a.top + t] = (float)(b.x - lse);
    out.place[row * a.top + t] = b.at == 0xffffffffu ? -1 : (int64_t)b.at;
  }
}

}  // namespace

// One part of one row. With parts == 1 it writes the row's results.
template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kThr) void k_scores(ScoreArgs a, ScoreOut out, int parts, Part* __restrict__ sums,
                                                 float* __restrict__ best, uint32_t* __restrict__ best_at) {
  constexpr int P = kPiece<T>;
  __shared__ Sums shared[kWaves];
  __shared__ Lists<TOP ? kWaves : 1> lists;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t);
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const T* x = row_at<T>(a, row);
  const int pieces = a.V / P, first = (int)((int64_t)pieces * part / parts), end = (int)((int64_t)pieces * (part + 1) / parts);
  Sums mine = kNothing;
  Few few;
  Best b;
  // The waves tell one another the last value that counts, when they come to it: late news lets more through, no less
  // (266 us for 273 over 4096 rows).
  __shared__ float lasts[kWaves];
  if constexpr (TOP) {
    if (lane == 0) lasts[w] = -INFINITY;
    __syncthreads();
  }
  float limit = -INFINITY;
  auto hear = [&]() {
    __hip_atomic_store(&lasts[w], b.last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
#pragma unroll
    for (int n = 0; n < kWaves; ++n)
      limit = fmaxf(limit, __hip_atomic_load(&lasts[n], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
  };
  auto take = [&](auto& v, uint32_t i, bool in) {
    constexpr int N = sizeof(v) / sizeof(v[0]);
    const float most = most_of(v);
    add<N, ENTROPY>(mine, few, v, most);
    if constexpr (TOP) offer<N>(b, v, most, i, in, limit, a.top, lane);
  };
  // A wave's turns: whole ones, of which the next is on its way, then piece by piece, with lanes past the end that have
  // nothing: a list belongs to all lanes.
  int i = first + 64 * w;
  auto load = [&](Raw<T>(&raw)[kTurn], int from) {
#pragma unroll
    for (int n = 0; n < kTurn; ++n) raw[n] = load_raw(x + (int64_t)(from + n * kThr + lane) * P);
  };
  constexpr int kWhole = (kTurn - 1) * kThr + 64;
  if (i + kWhole <= end) {
    Raw<T> next[kTurn];
    load(next, i);
    do {
      Raw<T> raw[kTurn];
#pragma unroll
      for (int n = 0; n < kTurn; ++n) raw[n] = next[n];
      const int after = i + kTurn * kThr;
      load(next, after + kWhole <= end ? after : i);
      if constexpr (TOP) hear();
#pragma unroll
      for (int n = 0; n < kTurn; ++n) {
        float v[P];
        values(v, raw[n]);
        take(v, (uint32_t)(i + n * kThr + lane) * P, true);
      }
      few.to(mine);
      i = after;
    } while (i + kWhole <= end);
  }
#pragma unroll 1
  for (; i < end; i += kThr) {
    const int p = i + lane;
    const Raw<T> raw = load_raw(x + (int64_t)min(p, end - 1) * P);
    float v[P];
    values(v, raw);
    if (p >= end)
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = -INFINITY;
    if constexpr (TOP) hear();
    take(v, (uint32_t)p * P, p < end);
    few.to(mine);
  }
  // values behind the last whole piece
  if (part == parts - 1 && w == kWaves - 1 && pieces * P < a.V) {
    const int p = pieces * P + lane;
    float v[1] = {p < a.V ? get(x + p) : -INFINITY};
    take(v, p, p < a.V);
    few.to(mine);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const Sums other = {__shfl_xor(mine.m, off, 64), __shfl_xor(mine.s, off, 64), __shfl_xor(mine.t, off, 64)};
    join(mine, other);
  }
  if (lane == 0) shared[w] = mine;
  if constexpr (TOP) join_lists(b, lists, w, lane);
  else __syncthreads();
  if (w) return;
  mine = shared[0];
#pragma unroll
  for (int n = 1; n < kWaves; ++n) join(mine, shared[n]);
  if (parts == 1) {
    finish<T, ENTROPY, TOP>(a, out, row, mine, b);
    return;
  }
  if (t == 0) sums[blockIdx.x] = {mine.s, mine.t, mine.m};
  if (TOP && t < a.top) {
    best[(size_t)blockIdx.x * a.top + t] = b.x;
    best_at[(size_t)blockIdx.x * a.top + t] = b.at;
  }
}

// The parts of one row, joined. A wave takes every kJoin-th part's list; without lists one wave is enough.
template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(64 * kJoin) void k_scores_join(ScoreArgs a, ScoreOut out, int parts,
                                                            const Part* __restrict__ sums,
                                                            const float* __restrict__ best,
                                                            const uint32_t* __restrict__ best_at) {
  __shared__ Lists<TOP ? kJoin : 1> lists;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t);
  const int64_t row = blockIdx.x;
  Best b;
  if constexpr (TOP) {
    for (int part = w; part < parts; part += kJoin) {
      const int n = 63 - lane;
      const int64_t at = (row * parts + part) * a.top + n;
      float x = -INFINITY;
      uint32_t i = 0xffffffffu;
      if (n < a.top) x = best[at], i = best_at[at];
      merge_sorted(b, x, i, lane);
    }
    join_lists(b, lists, w, lane);
  }
  if (w) return;
  // of at most 64 parts
  Sums mine = kNothing;
  if (lane < parts) {
    const Part x = sums[row * parts + lane];
    mine = {x.m, x.s, x.t};
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const Sums other = {__shfl_xor(mine.m, off, 64), __shfl_xor(mine.s, off, 64), __shfl_xor(mine.t, off, 64)};
    join(mine, other);
  }
  finish<T, ENTROPY, TOP>(a, out, row, mine, b);
}

// The gradient of one part of one row: the logits once more, with the row's maximum and sum from the forward, and as many
// bytes out; nothing else is kept from the forward, so that a loss takes no memory of the logits' size before it.
template <typename T>
__global__ __launch_bounds__(kThr) void k_scores_bwd(ScoreArgs a, int parts, const float* __restrict__ saved,
                                                     const float* __restrict__ entropy, const float* __restrict__ dlog,
                                                     const float* __restrict__ dentropy, T* __restrict__ dlogits) {
  constexpr int P = kPiece<T>;
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const T* x = row_at<T>(a, row);
  T* dx = dlogits + row * a.V;
  const int64_t token = a.tokens[row];
  const float m = saved[2 * row], s = saved[2 * row + 1], inv = 1.f / s;
  float dl = dlog && token >= 0 ? dlog[row] : 0.f;
  // what nobody asks about a token that there is not is no gradient, and the entropy does not depend on the token
  if (token >= a.V && dl != 0.f) dl = __builtin_nanf("");
  // -p (dl + dh (log p + H)), log p + H = z + base
  const float dh = dentropy ? dentropy[row] : 0.f, base = dentropy ? entropy[row] - logf(s) : 0.f;
  const float flat = -inv * (dl + dh * base), slope = -inv * dh;
  // rows that nothing is asked about have no gradient, also those without a distribution (padding, say)
  const bool asked = dl != 0.f || dh != 0.f;
  auto grad = [&](float v, int64_t i) {
    if (!asked) return 0.f;
    const float z = v - m;
    const float d = exp_of(z) * fmaf(slope, fmaxf(z, kGone), flat);  // where p is zero it is
    return i == token ? d + dl : d;
  };
  const int64_t pieces = a.V / P, first = pieces * part / parts, end = pieces * (part + 1) / parts;
  for (int64_t i = first + t; i < end; i += kTurn * kThr) {
    Raw<T> raw[kTurn];
#pragma unroll
    for (int n = 0; n < kTurn; ++n) raw[n] = load_raw(x + min(i + n * kThr, end - 1) * P);
#pragma unroll
    for (int n = 0; n < kTurn; ++n) {
      const int64_t p = i + n * kThr;
      if (p >= end) break;
      float v[P];
      values(v, raw[n]);
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = grad(v[e], p * P + e);
      store_raw(dx + p * P, v);
    }
  }
  const int64_t tail = pieces * P + t;
  if (part == parts - 1 && tail < a.V) put(dx + tail, grad(get(x + tail), tail));
}

namespace {
int score_parts(const ScoreArgs& a) {
  const int64_t rows = (int64_t)a.B * a.N;
  // Parts fill the GPU's 256 CUs four times, and a wave joins 64 parts at most. A part has a turn of the block's pieces
  // of fp32 logits or more; of 16-bit ones, whose pieces hold twice as many values, half a turn, so that few rows of them
  // (one of 151936: 49 parts of 387 pieces) go piece by piece, in more blocks. With twice or half as many blocks one row,
  // 48 and 2000 take the same within 1%.
  const int64_t most = std::max(1, a.V / (kThr * kTurn * 4));
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
        hipLaunchKernelGGL(second, dim3((unsigned)rows), dim3(a.top ? 64 * kJoin : 64), 0, st, a, out, parts, sums, best,
                           best_at);
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
