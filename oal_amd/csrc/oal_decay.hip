// Linear attention with decays for gfx950: chunked forward and backward over whole
// sequences, and the recurrence over single tokens.
//
//   S_t = a_t S_{t-1} + k_t v_t^T,  a_t = exp(g_t),  o_t = scale S_t^T q_t
//
// In chunks of 64 tokens, G the sums of g inside the chunk, S the state before it:
//   S' = e^(G_63) S + K^T (e^(G_63 - G) V)
//   O  = scale (e^G Q S + (exp(G_i - G_j) q_i.k_j)_(j <= i) V)
// and back, dS' the gradient of the state after the chunk:
//   dS = e^(G_63) dS' + scale (e^G Q)^T dO
//   dQ = scale (e^G dO S^T + (exp(G_i - G_j) dO_i.v_j)_(j <= i) K), dK and dV alike from dS'.
// A block walks a segment of chunks with the state in its accumulators; where there are too few
// units (batch and state heads) for the GPU, sequences are cut into segments, whose sums and a scan over them give the
// states that they start from. What makes the state and the decays' gradients is exact to fp32 whatever the tensors'
// type (oal_tile.hpp): a state is a sum over all tokens before it and is handed on in fp32.
//
// Decays enter as differences of sums, held in two floats (48 bits): a token that
// forgets everything (g of -inf, the first of a new text) leaves large sums whose differences still matter.
//
// 4 x 4096 tokens of 14/14/14 heads of 64, bf16, forward and backward: 199 us of kernels, of which the gradients are 106,
// the outputs 39, both sums 35, both scans 14. What has to be read and written takes 47 us at the rate of a large copy. What
// bounds it is the vector unit's work on operands (decays, splits into parts, fragments from LDS), 1800 instructions a
// wave and chunk in the backward, and waiting between phases that depend on one another: there the vector units
// are busy for 45 % of the time, the matrix units for 14 %, and waves wait for 42 % of theirs. A prompt of 32768 tokens, 7/7/14 heads: 91 us, copied in 35.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "oal_common.hpp"
#include "oal_decay.hpp"
#include "oal_tile.hpp"

namespace oal {

namespace {

constexpr int kThr = 256;
constexpr int kTile2 = 64 * 64;
// Smallest log-decay: exp of it is zero, and 64 of them leave the sums' differences exact.
constexpr double kLeast = -1e4;

// Of a chunk's tokens: log2 of the decay up to and with the token, in two parts; the decay since
// the chunk's start and until its end, and since and until those of its tile of 16 tokens. end: the chunk's decay in two
// parts, and its log2.
struct alignas(16) Decays {
  float hi[64], lo[64], since[64], until[64], head[64], tail[64], end[2];
  double log_end;
};
constexpr int kSlots = 4;  // chunks whose decays a block forms at once, a wave each

__device__ __forceinline__ f32x4 four(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
// The decays of a tile: from tokens r .. r + 3 to token (hi, lo), or with TO from it to them. Between tiles they
// are products of the tokens' own and one between the tiles' borders, an exponential where there would be four.
template <bool TO>
__device__ __forceinline__ f32x4 decays(const Decays& s, int r, int tile, bool same, float hi, float lo) {
  f32x4 y;
  if (same) {
    const f32x4 h = four(s.hi + r), l = four(s.lo + r);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      y[i] = __builtin_amdgcn_exp2f(TO ? (h[i] - hi) + (l[i] - lo) : (hi - h[i]) + (lo - l[i]));
  } else if constexpr (TO) {
    y = four(s.head + r) * __builtin_amdgcn_exp2f((s.hi[tile - 1] - hi) + (s.lo[tile - 1] - lo));
  } else {
    y = four(s.tail + r) * __builtin_amdgcn_exp2f((hi - s.hi[tile + 15]) + (lo - s.lo[tile + 15]));
  }
  return y;
}
// A number's parts: it is their sum to 48 bits.
__device__ __forceinline__ void in_two(double x, float (&y)[2]) {
  y[0] = (float)x;
  y[1] = (float)(x - (double)y[0]);
}
// What is forgotten is gone, NaN and infinities too: a decay of zero is no factor.
__device__ __forceinline__ f32x4 decayed(float by, const f32x4& x) { return by == 0.f ? f32x4{} : by * x; }
// y = e x + d, e in two parts: slow decays multiply for many chunks.
__device__ __forceinline__ float carry(const float (&e)[2], float x, float d) {
  return e[0] == 0.f ? d : fmaf(e[0], x, fmaf(e[1], x, d));
}

__device__ __forceinline__ float gate_at(const DecayArgs& a, int b, int h, int tok) {
  return static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + tok * a.g.n];
}

// A wave's running sums, the lane's own value with it: within rows of 16 lanes, then from rows to the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lanes(double x) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double running_sum_of_16(double x) {
  x += from_lanes<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8
  x += from_lanes<0x112, 0xf>(x);
  x += from_lanes<0x114, 0xf>(x);
  return x + from_lanes<0x118, 0xf>(x);
}
__device__ __forceinline__ double running_sum(double x) {
  x = running_sum_of_16(x);
  x += from_lanes<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x += from_lanes<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A wave: the decays of 64 tokens with log-decays gate.
__device__ __forceinline__ void form_decays(Decays& s, float gate, int lane) {
  const double x = running_sum((gate < kLeast ? kLeast : (double)gate) * 1.4426950408889634);
  const double end = lane_of(x, 63);
  float y[2];
  in_two(x, y);
  s.hi[lane] = y[0];
  s.lo[lane] = y[1];
  s.since[lane] = __builtin_amdgcn_exp2f(y[0] + y[1]);
  s.until[lane] = __builtin_amdgcn_exp2f((float)(end - x));
  // the last tokens of the tile before and of the own one
  const double b0 = lane_of(x, 15), b1 = lane_of(x, 31), b2 = lane_of(x, 47);
  const double before = lane < 16 ? 0.0 : lane < 32 ? b0 : lane < 48 ? b1 : b2;
  const double last = lane < 16 ? b0 : lane < 32 ? b1 : lane < 48 ? b2 : end;
  s.head[lane] = __builtin_amdgcn_exp2f((float)(x - before));
  s.tail[lane] = __builtin_amdgcn_exp2f((float)(last - x));
  if (lane == 0) {
    in_two(exp2(end), s.end);
    s.log_end = end;
  }
}

// A block's part of the walk: unit u = (b, h), chunks [first, last) of its segment, one after another or back.
struct Course {
  int u, b, h, seg, first, last;
  __device__ __forceinline__ Course(const DecayArgs& a, const DecaySegments& sg, int id) {
    seg = id % sg.count;
    u = id / sg.count;
    b = u / a.Hv;
    h = u % a.Hv;
    first = seg * sg.len;
    last = min(first + sg.len, a.NC);
  }
};
// Every kSlots chunks each wave forms the decays of one of the chunks that follow; their gates are on their way
// since the last time. Tokens past N decay nothing.
struct Gates {
  float next;
  __device__ __forceinline__ int token(const Course& x, int n, int step, int w, int lane) const {
    return 64 * ((step > 0 ? x.first : x.last - 1) + step * (n + w)) + lane;
  }
  __device__ __forceinline__ void fetch(const DecayArgs& a, const Course& x, int n, int step, int w, int lane) {
    next = gate_at(a, x.b, x.h, min(max(token(x, n, step, w, lane), 0), a.N - 1));
  }
  __device__ __forceinline__ void form(Decays (&dec)[kSlots], const DecayArgs& a, const Course& x, int n, int step, int w,
                                       int lane) {
    if (n % kSlots) return;
    if (n + w < x.last - x.first) form_decays(dec[w], token(x, n, step, w, lane) < a.N ? next : 0.f, lane);
    fetch(a, x, n + kSlots, step, w, lane);
  }
};

template <typename T>
__device__ __forceinline__ const T* rows_of(const Strided& s, int b, int h, int tok0) {
  return static_cast<const T*>(s.p) + b * s.b + h * s.h + (int64_t)tok0 * s.n;
}

// A window of memory from a base that the block shares, with 32-bit offsets (rows are less than 2^23 elements
// apart). What lies at kNowhere is read as zero and not written: loads and stores of rows past the last or columns
// past the width are none that a lane could skip, so that the ones in flight can be counted on every way.
constexpr uint32_t kNowhere = 0x80000000u;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
struct Window {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ explicit Window(const void* p)
      : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)(kNowhere - 16), 0x00027000)) {}
  __device__ __forceinline__ u32x4 load(uint32_t at) const { return __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0); }
  __device__ __forceinline__ void store(uint32_t at, const u32x4& x) const {
    __builtin_amdgcn_raw_buffer_store_b128(x, r, at, 0, 0);
  }
  __device__ __forceinline__ void store(uint32_t at, const u32x2& x) const {
    __builtin_amdgcn_raw_buffer_store_b64(x, r, at, 0, 0);
  }
};
// Four values to element `at`, or nowhere.
__device__ __forceinline__ void put4(const Window& w, const float*, bool in, uint32_t at, const f32x4& x) {
  w.store(in ? 4 * at : kNowhere, __builtin_bit_cast(u32x4, x));
}
__device__ __forceinline__ void put4(const Window& w, const uint16_t*, bool in, uint32_t at, const f32x4& x) {
  w.store(in ? 2 * at : kNowhere, u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])});
}
__device__ __forceinline__ void put4(const Window& w, const _Float16*, bool in, uint32_t at, const f32x4& x) {
  w.store(in ? 2 * at : kNowhere, __builtin_bit_cast(u32x2, __builtin_convertvector(x, f16x4)));
}
// Eight values of a row, or zeros, as they come.
template <typename T>
struct Eight {
  u32x4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const Window& from, bool in, uint32_t at) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = from.load(in ? at * (uint32_t)sizeof(T) + 16 * i : kNowhere);
  }
  template <int NP>
  __device__ __forceinline__ Frag<NP> parts() const {
    Frag<NP> f;
    if constexpr (NP == 1) {
      f.p[0] = __builtin_bit_cast(bf16x8, w[0]);
    } else {
      float x[8];
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e / 4][e % 4]);
      } else {
        typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
        const f16x8 v = __builtin_bit_cast(f16x8, w[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(v[e]);
      }
      f = split<NP>(x);
    }
    return f;
  }
};

// 64 rows of D values on their way to an LDS tile, by 256 threads; zeros for rows at and past `live` and columns from D.
template <int NP, typename T>
struct Coming {
  Eight<T> x[2];
  __device__ __forceinline__ void fetch(const T* base, uint32_t stride, int D, int live, int t) {
    const Window from(base);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = (t >> 3) + 32 * n, c = 8 * (t & 7);
      x[n].load(from, r < live && c < D, __umul24(r, stride) + c);
    }
  }
  __device__ __forceinline__ void store(Tile<NP>& s, int t) const {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const Frag<NP> f = x[n].template parts<NP>();
      __bf16* p = s.x + tile_at((t >> 3) + 32 * n, 8 * (t & 7));
#pragma unroll
      for (int e = 0; e < NP; ++e) *reinterpret_cast<bf16x8*>(p + e * kTileElems) = f.p[e];
    }
  }
};
// A token's row as operands of sums over its D values: 32 k + 8 g + j, on its way.
template <typename T>
struct ComingRow {
  Eight<T> x[2];
  __device__ __forceinline__ void fetch(const T* base, uint32_t stride, int D, int live, int row, int g) {
    const Window from(base);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      x[k].load(from, row < live && 32 * k + 8 * g < D, __umul24(row, stride) + 32 * k + 8 * g);
  }
};

// Row `row` of a tile as the accumulators of a product with it have it: values 16 m + 4 g + i.
template <int NP>
__device__ __forceinline__ f32x4 own_values(const Tile<NP>& s, int row, int m, int lane) {
  f32x4 x = {};
#pragma unroll
  for (int e = NP - 1; e >= 0; --e)
    x += __builtin_convertvector(
        *reinterpret_cast<const bf16x4*>(s.x + e * kTileElems + tile_at(row, 16 * m + 4 * (lane >> 4))), f32x4);
  return x;
}

// An accumulator tile in parts: two of them are the operand of a sum over their 32 rows (perm order).
template <int N>
struct Half {
  bf16x4 p[N];
};
template <int N>
__device__ __forceinline__ Half<N> half_of(const f32x4& x) {
  Half<N> h;
  float v[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int e = 0; e < N; ++e) {
    h.p[e] = __builtin_bit_cast(bf16x4, pack4(v));
    if (e + 1 < N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] -= static_cast<float>(h.p[e][i]);
    }
  }
  return h;
}
template <int N>
__device__ __forceinline__ Frag<N> both(const Half<N>& a, const Half<N>& b) {
  Frag<N> f;
#pragma unroll
  for (int e = 0; e < N; ++e) f.p[e] = __builtin_shufflevector(a.p[e], b.p[e], 0, 1, 2, 3, 4, 5, 6, 7);
  return f;
}

// Columns c0 .. of a tile of 64 rows, read by rows 32 s + 8 g + j, each row scaled: an operand of UP parts, exact to fp32
// if three.
template <int UP, int NP>
__device__ __forceinline__ Frag<UP> scaled_col(const Tile<NP>& s, int c0, int half, int lane, const float* by, float scale) {
  const Frag<NP> f = col_frag(s, c0, half, lane);
  const int g = lane >> 4;
  const f32x4 b0 = scale * four(by + 32 * half + 8 * g), b1 = scale * four(by + 32 * half + 8 * g + 4);
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = 0.f;
#pragma unroll
    for (int x = NP - 1; x >= 0; --x) v[j] += static_cast<float>(f.p[x][j]);
    v[j] *= j < 4 ? b0[j] : b1[j - 4];
  }
  return split<UP>(v);
}

// Sums over a row of 16 lanes, in all of them.
__device__ __forceinline__ float sum_of_16(float x) {
  auto add = [&](auto how) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(how)::value, 0xf, 0xf, true));
  };
  add(std::integral_constant<int, 0x128>());  // row_ror:8, 4, 2, 1
  add(std::integral_constant<int, 0x124>());
  add(std::integral_constant<int, 0x122>());
  add(std::integral_constant<int, 0x121>());
  return x;
}
// The sum of what the lane groups before have in this column.
__device__ __forceinline__ float groups_before(float x, int g) {
  const float up = __shfl_up(x, 16, 64), a = g >= 1 ? up : 0.f;
  const float next = __shfl_up(a, 16, 64), b = a + (g >= 2 ? next : 0.f);
  const float last = __shfl_up(a, 32, 64);
  return b + (g == 3 ? last : 0.f);
}
// Sums over the lane groups of one column: of a in group 0, b in 1, c in 2, d in 3.
__device__ __forceinline__ float group_sums(float a, float b, float c, float d, int g) {
  const bool high = g & 2, odd = g & 1;
  const float x = (high ? c : a) + __shfl_xor(high ? a : c, 32, 64), y = (high ? d : b) + __shfl_xor(high ? b : d, 32, 64);
  return (odd ? y : x) + __shfl_xor(odd ? x : y, 16, 64);
}

// Nothing moves over it: operands of later products, loaded early, would not fit the registers.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// What follows from it is computed here: kept from before a loop, all the addresses in LDS would not fit either.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Parts of the scores inside a chunk. bf16 ones in two, off by 2^-17, as float16 ones, so that a result is rounded once, to
// its own type: in one part bf16 results were 2.2e-3 off where a rounding is 1.7e-3 (4 x 4096 tokens, forward and
// backward, 192 us for 199); three parts take 9 us more.
template <typename T>
constexpr int kScoreParts = kPartsOf<T> == 1 ? 2 : kPartsOf<T>;
// Parts of the states that 16-bit results read: two too. In one part bf16 outputs were 1.9e-3 off (32768 tokens,
// k_decay_out 51 us for 56); three parts leave room for three blocks a CU in place of four (67 us).
template <typename T>
constexpr int kStateParts = kPartsOf<T> == 1 ? 2 : kPartsOf<T>;

// A state in accumulators, four tiles of a wave's 16 columns: S[m][i] is row 16 m + 4 g + i of column 16 w + c.
typedef f32x4 State[4];
// x += A^T (by B) over the rows of two tiles, A's columns the rows of x and B's 16 w .. the wave's columns.
template <int UP, int NP>
__device__ __forceinline__ void add_outer(State& x, const Tile<NP>& A, const Tile<NP>& B, const float* by, float scale,
                                          int w, int lane) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    phase();
    const Frag<UP> b = scaled_col<UP>(B, 16 * w, s, lane, by, scale);
#pragma unroll
    for (int m = 0; m < 4; ++m) x[m] = mma(col_frag(A, 16 * m, s, lane), b, x[m]);
  }
  phase();
}
// Over a few chunks one part of their decays does (2^-25 each); over many two.
__device__ __forceinline__ void decay_state(State& x, const float (&end)[2], const DecaySegments& sg) {
#pragma unroll
  for (int m = 0; m < 4; ++m) x[m] = decayed(end[0] + (sg.len > 8 ? 0.f : end[1]), x[m]);
  if (sg.len > 8) {
    const float more = end[0] == 0.f ? 0.f : end[1] / end[0];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[m][i] = fmaf(more, x[m][i], x[m][i]);
  }
}
// The state's columns as rows of a tile: four consecutive rows of the state at once.
template <int NP>
__device__ __forceinline__ void put_state(Tile<NP>& s, const State& x, int w, int lane) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const Half<NP> h = half_of<NP>(x[m]);
#pragma unroll
    for (int e = 0; e < NP; ++e)
      *reinterpret_cast<bf16x4*>(s.x + e * kTileElems + tile_at(16 * w + (lane & 15), 16 * m + 4 * (lane >> 4))) = h.p[e];
  }
}
// A state [rows][cols] in memory: TURNED where the accumulators' rows are its columns. Past its edges zero.
template <bool TURNED>
__device__ __forceinline__ void load_state(State& x, const float* p, int rows, int cols, int w, int lane) {
  const int own = 16 * w + (lane & 15);
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int r = 16 * m + 4 * (lane >> 4);
    x[m] = f32x4{};
    if (!p) continue;
    if constexpr (TURNED) {
      if (own < rows && r < cols) x[m] = load4(p + own * cols + r);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i < rows && own < cols) x[m][i] = p[(r + i) * cols + own];
    }
  }
}
template <bool TURNED>
__device__ __forceinline__ void store_state(const State& x, float* p, int rows, int cols, int w, int lane) {
  const int own = 16 * w + (lane & 15);
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const int r = 16 * m + 4 * (lane >> 4);
    if constexpr (TURNED) {
      if (own < rows && r < cols) store4(p + own * cols + r, x[m]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r + i < rows && own < cols) p[(r + i) * cols + own] = x[m][i];
    }
  }
}
// A whole state in memory, its columns the accumulators' rows.
__device__ __forceinline__ void load_tile(State& x, const float* p, int w, int lane) {
#pragma unroll
  for (int m = 0; m < 4; ++m) x[m] = load4(p + (16 * w + (lane & 15)) * 64 + 16 * m + 4 * (lane >> 4));
}
__device__ __forceinline__ void store_tile(const State& x, float* p, int w, int lane) {
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) p[(16 * m + 4 * (lane >> 4) + i) * 64 + 16 * w + (lane & 15)] = x[m][i];
}
// What a segment starts from: the states of the scan, or the call's own where there is but one segment.
struct From {
  const float* p;
  int rows, cols;
  __device__ __forceinline__ const float* of(const DecaySegments& sg, const Course& x) const {
    return p ? p + ((size_t)x.u * sg.count + x.seg) * rows * cols : nullptr;
  }
};

}  // namespace

// What a segment adds to the state, or (BACK) what its outputs ask of the state before it, over a state's
// output heads: k, v or q, dO of its chunks, one after another; and its decay. 17 us over 4 x 4096 tokens (59 MB). The next
// chunk is on its way while one is worked on; with the next two there the registers leave three waves a SIMD for
// four, and training takes 187 us for 185.
template <typename T, bool BACK>
__global__ __launch_bounds__(kThr) void k_decay_sum(DecayArgs a, DecaySegments sg, const T* __restrict__ dout,
                                                    float* __restrict__ G, float* __restrict__ D) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> A, B;
  __shared__ Decays dec[kSlots];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t);
  const Course x(a, sg, blockIdx.x);
  const int each = BACK ? a.H / a.Hv : 1, o0 = x.h * each, count = (x.last - x.first) * each;
  Coming<NP, T> ai, bi;
  auto fetch = [&](int i) {
    const int n = i / each, o = o0 + i % each, ch = BACK ? x.last - 1 - n : x.first + n;
    const int tok0 = 64 * ch, live = min(64, a.N - tok0);
    if constexpr (BACK) {
      ai.fetch(rows_of<T>(a.q, x.b, o / (a.H / a.Hq), tok0), a.q.n, a.D, live, t);
      bi.fetch(dout + (((size_t)x.b * a.H + o) * a.N + tok0) * a.DV, a.DV, a.DV, live, t);
    } else {
      ai.fetch(rows_of<T>(a.k, x.b, x.h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
      bi.fetch(rows_of<T>(a.v, x.b, x.h, tok0), a.v.n, a.DV, live, t);
    }
  };
  State s = {};
  double log = 0;
  Gates gates;
  gates.fetch(a, x, 0, BACK ? -1 : 1, w, lane);
  fetch(0);
  for (int i = 0; i < count; ++i) {
    const int n = i / each, ch = BACK ? x.last - 1 - n : x.first + n;
    if (i) lds_sync();
    if (i % each == 0) gates.form(dec, a, x, n, BACK ? -1 : 1, w, lane);
    ai.store(A, t);
    bi.store(B, t);
    lds_sync();
    fetch(min(i + 1, count - 1));
    const Decays& d = dec[n % kSlots];
    if (i % each == 0) {
      decay_state(s, d.end, sg);
      log += d.log_end;
    }
    add_outer<3>(s, A, B, BACK ? d.since : d.until, BACK ? a.scale : 1.f, w, lane);
  }
  store_tile(s, D + (size_t)blockIdx.x * kTile2, w, lane);
  float y[2];
  in_two(exp2(log), y);
  if (t == 0) G[2 * blockIdx.x] = y[0], G[2 * blockIdx.x + 1] = y[1];
}

// S' = e S + D over the segments, or back over them; what a segment adds is replaced by the state
// that it starts from (back: whose gradient it takes). A value per thread, the next ones on their way: 14 us
// for both scans over 4 x 4096 tokens, 16 and 8 segments of 56 states (15 and 7 MB in and out again).
struct Scan {
  const float* G;
  float* S;           // [U][segments][64][64]
  const float* init;  // [U][rows][cols] (null: zero)
  float* end;         // the same: the state after the last (null: not wanted)
  int count, rows, cols;
  bool back;
};
constexpr int kAhead = 8;
__global__ __launch_bounds__(kThr) void k_decay_scan(Scan a) {
  const int x = blockIdx.x * kThr + threadIdx.x, u = x / kTile2, i = x % kTile2, row = i / 64, col = i % 64;
  float s = 0.f;
  const bool held = row < a.rows && col < a.cols;
  const size_t slot = ((size_t)u * a.rows + row) * a.cols + col;
  if (a.init && held) s = a.init[slot];
  for (int n0 = 0; n0 < a.count; n0 += kAhead) {
    float d[kAhead], e[kAhead][2];
    auto at = [&](int n) { return (size_t)u * a.count + (a.back ? a.count - 1 - n : n); };
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const size_t k = at(min(n0 + n, a.count - 1));
      d[n] = a.S[k * kTile2 + i];
      e[n][0] = a.G[2 * k], e[n][1] = a.G[2 * k + 1];
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      if (n0 + n >= a.count) break;
      a.S[at(n0 + n) * kTile2 + i] = s;
      s = carry(e[n], s, d[n]);
    }
  }
  if (a.end && held) a.end[slot] = s;
}

// The outputs of one segment for `each` output heads of a state head, chunk by chunk, with the state in
// accumulators and, as bf16 parts (kStateParts), in LDS. Outputs are transposed: a wave's 16 queries
// are the columns, so the scores are an operand of the product with V as they are.
// UP: parts of what the state takes on, three where it goes on to the caller or (states: kept before every
// chunk) to the backward, two, off by 2^-17 as what outputs read of it, where no further than the segment's own outputs (32768 tokens: 56 us
// for 62). In training 39 us over 4 x 4096 tokens, 117 MB of heads and 59 MB of states (4.5 TB/s).
template <typename T, int UP>
__global__ __launch_bounds__(kThr, kPartsOf<T> == 1 ? 4 : 2) void k_decay_out(DecayArgs a, DecaySegments sg, int each,
                                                                              From from, T* __restrict__ out,
                                                                              float* __restrict__ final_state,
                                                                              float* __restrict__ states) {
  constexpr int NP = kPartsOf<T>, SP = kScoreParts<T>;
  __shared__ Tile<NP> K, V;
  __shared__ Tile<kStateParts<T>> S;  // rows: values
  __shared__ Decays dec[kSlots];
  int t = threadIdx.x, lane = t & 63;
  const int w = wave_of(t), g = lane >> 4, c = lane & 15, own = 16 * w + c;
  const int rep = a.H / a.Hv, parts = (rep + each - 1) / each, part = blockIdx.x % parts;
  const Course x(a, sg, blockIdx.x / parts);
  const int o0 = x.h * rep + part * each, o1 = min(o0 + each, (x.h + 1) * rep);
  State s;
  load_state<false>(s, from.of(sg, x), from.rows, from.cols, w, lane);
  Coming<NP, T> ki, vi;
  ComingRow<T> next;
  auto fetch = [&](int ch) {
    const int tok0 = 64 * ch, live = min(64, a.N - tok0);
    ki.fetch(rows_of<T>(a.k, x.b, x.h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
    vi.fetch(rows_of<T>(a.v, x.b, x.h, tok0), a.v.n, a.DV, live, t);
  };
  auto fetch_q = [&](int ch, int o) {
    next.fetch(rows_of<T>(a.q, x.b, o / (a.H / a.Hq), 64 * ch), a.q.n, a.D, a.N - 64 * ch, own, g);
  };
  Gates gates;
  gates.fetch(a, x, 0, 1, w, lane);
  fetch(x.first);
  fetch_q(x.first, o0);
  for (int ch = x.first; ch < x.last; ++ch) {
    const int n = ch - x.first, tok0 = 64 * ch, live = min(64, a.N - tok0);
    lane = here(lane), t = here(t);
    if (n) lds_sync();
    gates.form(dec, a, x, n, 1, w, lane);
    ki.store(K, t);
    vi.store(V, t);
    put_state(S, s, w, lane);
    if (states && part == 0) store_tile(s, states + ((size_t)x.u * a.NC + ch) * kTile2, w, lane);
    lds_sync();
    fetch(min(ch + 1, x.last - 1));
    const Decays& d = dec[n % kSlots];
    const float since = a.scale * d.since[own], hi = d.hi[own], lo = d.lo[own];
    int o = o0;
    do {  // once at least: what is in flight behind it can be counted
      lane = here(lane);
      const Frag<NP> qf[2] = {next.x[0].template parts<NP>(), next.x[1].template parts<NP>()};
      fetch_q(o + 1 < o1 ? ch : min(ch + 1, x.last - 1), o + 1 < o1 ? o + 1 : o0);
      Half<SP> p[4] = {};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m > w) continue;
        f32x4 y = {};
#pragma unroll
        for (int k = 0; k < 2; ++k) y = mma(row_frag(K, 16 * m, k, lane), qf[k], y);
        y *= a.scale * decays<false>(d, 16 * m + 4 * g, 16 * m, m == w, hi, lo);
        if (m == w)
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = 4 * g + i <= c ? y[i] : 0.f;
        p[m] = half_of<SP>(y);
      }
      phase();
      const Frag<SP> p0 = both(p[0], p[1]), p1 = both(p[2], p[3]);
      const Window dst(out + (((size_t)x.b * a.H + o) * a.N + tok0) * a.DV);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        f32x4 y = {};
#pragma unroll
        for (int k = 0; k < 2; ++k) y = mma(row_frag(S, 16 * m, k, lane), qf[k], y);
        y = decayed(since, y);
        y = mma(col_frag_perm(V, 16 * m, 0, lane), p0, y);
        if (w >= 2) y = mma(col_frag_perm(V, 16 * m, 1, lane), p1, y);
        put4(dst, out, own < live && 16 * m + 4 * g < a.DV, __umul24(own, a.DV) + 16 * m + 4 * g, y);
      }
    } while (++o < o1);
    if (ch + 1 < x.last || UP == 3) {
      decay_state(s, d.end, sg);
      add_outer<UP>(s, K, V, d.until, 1.f, w, lane);
    }
  }
  if (UP == 3 && final_state && x.last == a.NC && part == 0)
    store_state<false>(s, final_state + (size_t)x.u * a.D * a.DV, a.D, a.DV, w, lane);
}

// ---------------------------------------------------------------------------
// Backward, with D_ij = scale exp(G_i - G_j) (j <= i) in a chunk, S before it and dS' behind it:
//   dq_i = scale e^(G_i) S dO_i + sum_j D_ij (dO_i.v_j) k_j     (per output head)
//   dk_j = e^(G_63 - G_j) dS' v_j + sum_i D_ij (dO_i.v_j) q_i
//   dv_j = e^(G_63 - G_j) dS'^T k_j + sum_i D_ij (q_i.k_j) dO_i
//   dg_t = sum over all pairs j < t <= i of what passes from j to i: with M_ij = D_ij (q_i.k_j) (dO_i.v_j),
//     a_i = scale e^(G_i) q_i.(S dO_i), s_j = e^(G_63 - G_j) k_j.(dS' v_j),
//     dg_t = sum_(j < t <= i) M_ij + sum_(i >= t) a_i + sum_(j < t) s_j + e^(G_63) <S, dS'>
//   and no pair that t is not between: where its decay is strong, those are larger than what is asked for by any factor.
//   So of the pairs of the tiles m <= w of 16 tokens, t in tile T, those with m < T = w are summed over j by query, from t
//   on; those with m = T < w over i by key, up to t; those of m < T < w whole; those of m = T = w one by one.
// A block walks back with dS' in its accumulators; S the forward has kept. Both take turns in one tile of LDS. All
// products are transposed: a wave's 16 tokens are the columns. dg
// sees all 24 bits of the states, in three parts of X, and so do dq and dk; dv takes kStateParts.
// 106 us over 4 x 4096 tokens, 448 blocks at two a CU with all their registers (bf16: ten of them in scratch): 64 CUs have
// but one. dg as a difference of sums over all pairs took 96 us and left noise of 1e-7 of the largest sum.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThr, kPartsOf<T> == 1 ? 2 : 1) void k_decay_bwd(
    DecayArgs a, DecaySegments sg, From from, const T* __restrict__ dout, const float* __restrict__ states,
    T* __restrict__ dq, float* __restrict__ dqh, T* __restrict__ dk, float* __restrict__ dkh, T* __restrict__ dv,
    float* __restrict__ dg, double* __restrict__ dgsum, float* __restrict__ dstate) {
  constexpr int NP = kPartsOf<T>, SP = kScoreParts<T>;
  __shared__ Tile<NP> K, V, Q, O;
  __shared__ Tile<3> X;  // rows: keys' dimensions
  __shared__ Decays dec[kSlots];
  __shared__ float ss[2][64], ends[2][4];
  // a_i; M of a query with the keys of the tiles before its own, of the first, of the first two; of a key with the queries
  // of the tiles behind its own; of the pairs around a token in its tile
  __shared__ double ofq[2][4][64], ofk[2][64], ofd[2][64];
  int t = threadIdx.x, lane = t & 63;
  const int w = wave_of(t), g = lane >> 4, c = lane & 15, own = 16 * w + c;
  const Course x(a, sg, blockIdx.x);
  const int each = a.H / a.Hv, o0 = x.h * each;
  State s;  // the gradient of the state; rows: values, columns: keys' dimensions
  load_state<true>(s, from.of(sg, x), from.rows, from.cols, w, lane);
  Coming<NP, T> ki, vi, qi, oi;
  auto krows = [&](int ch) { return rows_of<T>(a.k, x.b, x.h / (a.Hv / a.Hk), 64 * ch); };
  auto qrows = [&](int ch, int o) { return rows_of<T>(a.q, x.b, o / (a.H / a.Hq), 64 * ch); };
  auto fetch = [&](int ch, int o) {
    const int tok0 = 64 * ch, live = min(64, a.N - tok0);
    qi.fetch(qrows(ch, o), a.q.n, a.D, live, t);
    oi.fetch(dout + (((size_t)x.b * a.H + o) * a.N + tok0) * a.DV, a.DV, a.DV, live, t);
  };
  auto fetch_k = [&](int ch) {
    const int live = min(64, a.N - 64 * ch);
    ki.fetch(krows(ch), a.k.n, a.D, live, t);
    vi.fetch(rows_of<T>(a.v, x.b, x.h, 64 * ch), a.v.n, a.DV, live, t);
  };
  State before;
  auto fetch_state = [&](int ch) {
    load_tile(before, states + ((size_t)x.u * a.NC + ch) * kTile2, w, lane);
  };
  Gates gates;
  gates.fetch(a, x, 0, -1, w, lane);
  fetch_k(x.last - 1);
  fetch(x.last - 1, o0);
  fetch_state(x.last - 1);
  for (int ch = x.last - 1; ch >= x.first; --ch) {
    const int n = x.last - 1 - ch, tok0 = 64 * ch, live = min(64, a.N - tok0), turn = n & 1;
    lane = here(lane), t = here(t);
    gates.form(dec, a, x, n, -1, w, lane);
    ki.store(K, t);
    vi.store(V, t);
    qi.store(Q, t);
    oi.store(O, t);
    put_state(X, s, w, lane);
    lds_sync();
    fetch_k(max(ch - 1, x.first));
    const Decays& d = dec[n % kSlots];
    const float hi = d.hi[own], lo = d.lo[own], since = a.scale * d.since[own];
    f32x4 wk[4], wv[4];
    float passed = 0.f;  // s_j
    {
      const Frag<NP> kf[2] = {row_frag(K, 16 * w, 0, lane), row_frag(K, 16 * w, 1, lane)};
      const Frag<NP> vf[2] = {row_frag(V, 16 * w, 0, lane), row_frag(V, 16 * w, 1, lane)};
      const float until = d.until[own];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        f32x4 y = {}, z = {};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y = mma(row_frag(X, 16 * m, i, lane), vf[i], y);
          z = mma(col_frag<kStateParts<T>>(X, 16 * m, i, lane), kf[i], z);
        }
        wk[m] = decayed(until, y);
        wv[m] = decayed(until, z);
        const f32x4 k = own_values(K, own, m, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) passed += k[i] * wk[m][i];
      }
    }
    // the gradient of the state before the chunk, and what passes the whole chunk
    decay_state(s, d.end, sg);
    float through = 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) through += before[m][i] * s[m][i];
    through = d.end[0] == 0.f ? 0.f : wave_sum(through);
    lds_sync();
    put_state(X, before, w, lane);
    fetch_state(max(ch - 1, x.first));
    int o = o0;
    do {
      lane = here(lane), t = here(t);
      if (o > o0) {
        lds_sync();
        qi.store(Q, t);
        oi.store(O, t);
      }
      lds_sync();
      fetch(o + 1 < o0 + each ? ch : max(ch - 1, x.first), o + 1 < o0 + each ? o + 1 : o0);
      // of the head; their sums over heads are in 64 bits
      auto add = [&](double& sum, float x) { sum = x + (o > o0 ? sum : 0.0); };
      {
        float a_i = 0.f, near = 0.f, first = 0.f, two = 0.f;
        // queries: own
        const Frag<NP> qf[2] = {row_frag(Q, 16 * w, 0, lane), row_frag(Q, 16 * w, 1, lane)};
        const Frag<NP> of[2] = {row_frag(O, 16 * w, 0, lane), row_frag(O, 16 * w, 1, lane)};
        Half<SP> p[4] = {};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (m > w) continue;
          f32x4 y = {}, qk = {};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            y = mma(row_frag(V, 16 * m, i, lane), of[i], y);
            qk = mma(row_frag(K, 16 * m, i, lane), qf[i], qk);
          }
          y *= a.scale * decays<false>(d, 16 * m + 4 * g, 16 * m, m == w, hi, lo);
          if (m == w) {
            // pairs (j, own query) summed over the keys before 4 g + i, then over the queries from there on
            float x[4], before[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              x[i] = 4 * g + i < c ? y[i] * qk[i] : 0.f;
              y[i] = 4 * g + i <= c ? y[i] : 0.f;
              before[i] = i ? before[i - 1] + x[i - 1] : 0.f;
            }
            const float less = groups_before(before[3] + x[3], g);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = sum_of_16(4 * g + i <= c ? less + before[i] : 0.f);
            if (c < 4) add(ofd[turn][16 * w + 4 * g + c], c == 0 ? x[0] : c == 1 ? x[1] : c == 2 ? x[2] : x[3]);
          } else {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) x += y[i] * qk[i];
            near += x;
            if (m == 0 && w >= 2) first += x;
            if (m <= 1 && w == 3) two += x;
          }
          p[m] = half_of<SP>(y);
        }
        const Frag<SP> p0 = both(p[0], p[1]), p1 = both(p[2], p[3]);
        const size_t at = (((size_t)x.b * a.H + o) * a.N + tok0) * a.D;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          f32x4 y = {};
#pragma unroll
          for (int i = 0; i < 2; ++i) y = mma(row_frag(X, 16 * m, i, lane), of[i], y);
          y = decayed(since, y);
          const f32x4 q = own_values(Q, own, m, lane);
#pragma unroll
          for (int i = 0; i < 4; ++i) a_i += q[i] * y[i];
          y = mma(col_frag_perm(K, 16 * m, 0, lane), p0, y);
          if (w >= 2) y = mma(col_frag_perm(K, 16 * m, 1, lane), p1, y);
          const bool in = own < live && 16 * m + 4 * g < a.D;
          const uint32_t to = __umul24(own, a.D) + 16 * m + 4 * g;
          if (dqh)
            put4(Window(dqh + at), dqh, in, to, y);
          else
            put4(Window(dq + at), dq, in, to, y);
        }
        // each lane group has the sum of another one
        add(ofq[turn][g][own], group_sums(a_i, near, first, two, g));
      }
      phase();
      {
        // keys: own
        float behind = 0.f;
        const Frag<NP> kf[2] = {row_frag(K, 16 * w, 0, lane), row_frag(K, 16 * w, 1, lane)};
        const Frag<NP> vf[2] = {row_frag(V, 16 * w, 0, lane), row_frag(V, 16 * w, 1, lane)};
        Half<SP> p[4] = {}, r[4] = {};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (m < w) continue;
          f32x4 qk = {}, ov = {};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ov = mma(row_frag(O, 16 * m, i, lane), vf[i], ov);
            qk = mma(row_frag(Q, 16 * m, i, lane), kf[i], qk);
          }
          f32x4 e = a.scale * decays<true>(d, 16 * m + 4 * g, 16 * m, m == w, hi, lo);
          if (m == w)
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = c <= 4 * g + i ? e[i] : 0.f;
          ov *= e;
#pragma unroll
          for (int i = 0; i < 4; ++i) behind += m > w ? ov[i] * qk[i] : 0.f;
          p[m] = half_of<SP>(ov);
          r[m] = half_of<SP>(e * qk);
        }
        const Frag<SP> p0 = both(p[0], p[1]), p1 = both(p[2], p[3]), r0 = both(r[0], r[1]), r1 = both(r[2], r[3]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (w < 2) {
            wk[m] = mma(col_frag_perm(Q, 16 * m, 0, lane), p0, wk[m]);
            wv[m] = mma(col_frag_perm(O, 16 * m, 0, lane), r0, wv[m]);
          }
          wk[m] = mma(col_frag_perm(Q, 16 * m, 1, lane), p1, wk[m]);
          wv[m] = mma(col_frag_perm(O, 16 * m, 1, lane), r1, wv[m]);
        }
        behind = group_sum(behind);
        if (g == 0) add(ofk[turn][own], behind);
      }
      if (ch > x.first || (dstate && sg.count == 1)) add_outer<3>(s, O, Q, d.since, a.scale, w, lane);
    } while (++o < o0 + each);
    const size_t at = (size_t)x.u * a.N + tok0;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int e = 16 * m + 4 * g;
      const uint32_t to = __umul24(own, a.D) + e;
      if (dkh)
        put4(Window(dkh + at * a.D), dkh, own < live && e < a.D, to, wk[m]);
      else
        put4(Window(dk + at * a.D), dk, own < live && e < a.D, to, wk[m]);
      put4(Window(dv + at * a.DV), dv, own < live && e < a.DV, __umul24(own, a.DV) + e, wv[m]);
    }
    passed = group_sum(passed);
    if (g == 0) ss[turn][own] = passed;
    if (lane == 0) ends[turn][w] = through;
    lds_sync();
    // one wave, another for each chunk; the next but one chunk writes these places again, behind a barrier
    if (w == n % 4) {
      // sums from a token on are running sums from the last one back
      const int back = 63 - lane;
      const double from = running_sum(ofq[turn][0][back]) + running_sum_of_16(ofq[turn][1][back]);
      const double until = running_sum(lane ? (double)ss[turn][lane - 1] : 0.0) +
                           running_sum_of_16(c ? ofk[turn][lane - 1] : 0.0);
      // over a whole tile; those that none passes have zeros
      const float over1 = wave_sum((float)ofq[turn][2][lane]), over2 = wave_sum((float)ofq[turn][3][lane]);
      double y = __shfl(from, back, 64) + until + ofd[turn][lane] + (g == 1 ? over1 : g == 2 ? over2 : 0.f) +
                 (((double)ends[turn][0] + ends[turn][1]) + ((double)ends[turn][2] + ends[turn][3]));
      if (lane >= live) y = 0;
      if (dgsum) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) y += __shfl_xor(y, off, 64);
        if (lane == 0) dgsum[(size_t)x.u * a.NC + ch] = y;
      } else if (lane < live) {
        dg[(size_t)x.u * a.N + tok0 + lane] = (float)y;
      }
    }
  }
  if (dstate && sg.count == 1) store_state<true>(s, dstate + (size_t)x.u * a.D * a.DV, a.D, a.DV, w, lane);
}

// The gradient of a head's one decay: its chunks' sums over the batch, a block per head.
__global__ __launch_bounds__(kThr) void k_decay_gate_sum(const double* __restrict__ src, int B, int Hv, int NC,
                                                         float* __restrict__ dg) {
  __shared__ double sum[kThr];
  const int t = threadIdx.x, h = blockIdx.x;
  double x = 0;
  for (int64_t i = t; i < (int64_t)B * NC; i += kThr) x += src[((i / NC) * Hv + h) * NC + i % NC];
  sum[t] = x;
  __syncthreads();
  for (int n = kThr / 2; n > 0; n >>= 1) {
    if (t < n) sum[t] += sum[t + n];
    __syncthreads();
  }
  if (t == 0) dg[h] = (float)sum[0];
}

// ---------------------------------------------------------------------------
// The recurrence itself, for single tokens: a block per state head holds the
// state, 4 x 4 values per thread, for all N tokens and writes it back.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThr) void k_decay_step(DecayStepArgs a) {
  __shared__ float sum[2][4][64];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t);
  const int u = blockIdx.x, b = u / a.Hv, h = u % a.Hv;
  const int d0 = 4 * (t >> 4), c0 = 4 * (t & 15);
  float* state = a.state + (size_t)u * a.Dk * a.Dv;
  // pieces of four are whole and aligned
  const bool fours = a.Dv % 4 == 0 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
  float s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float4 v = make_float4(0, 0, 0, 0);
    const float* p = state + (d0 + i) * a.Dv + c0;
    if (d0 + i < a.Dk && c0 < a.Dv) {
      if (fours)
        v = *reinterpret_cast<const float4*>(p);
      else
        v = make_float4(p[0], c0 + 1 < a.Dv ? p[1] : 0.f, c0 + 2 < a.Dv ? p[2] : 0.f, c0 + 3 < a.Dv ? p[3] : 0.f);
    }
    s[i][0] = v.x, s[i][1] = v.y, s[i][2] = v.z, s[i][3] = v.w;
  }
  const T* k = static_cast<const T*>(a.k.p) + b * a.k.b + (h / (a.Hv / a.Hk)) * a.k.h;
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.b + h * a.v.h;
  const int each = a.H / a.Hv;
  int turn = 0;
  for (int n = 0; n < a.N; ++n) {
    const float decay = expf(static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + n * a.g.n]);
    if (decay == 0.f) {  // gone, NaN and infinities too
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    }
    float vc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vc[j] = c0 + j < a.Dv ? get(v + n * a.v.n + c0 + j) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float ki = d0 + i < a.Dk ? get(k + n * a.k.n + d0 + i) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = fmaf(ki, vc[j], decay * s[i][j]);
    }
    for (int o = h * each; o < (h + 1) * each; ++o, turn ^= 1) {
      const T* q = static_cast<const T*>(a.q.p) + b * a.q.b + (o / (a.H / a.Hq)) * a.q.h + n * a.q.n;
      float y[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float qi = d0 + i < a.Dk ? get(q + d0 + i) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fmaf(qi, s[i][j], y[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = group_sum(y[j]);
      // the sums of a turn are read before the next but one writes over them
      if (lane < 16)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[turn][w][c0 + j] = y[j];
      lds_sync();
      T* out = static_cast<T*>(a.out) + (((size_t)b * a.H + o) * a.N + n) * a.Dv;
      if (t < a.Dv)
        put(out + t, a.scale * ((sum[turn][0][t] + sum[turn][1][t]) + (sum[turn][2][t] + sum[turn][3][t])));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float* p = state + (d0 + i) * a.Dv + c0;
    if (d0 + i >= a.Dk || c0 >= a.Dv) continue;
    if (fours) {
      *reinterpret_cast<float4*>(p) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + j < a.Dv) p[j] = s[i][j];
    }
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
namespace {
struct Room {
  char* base;
  size_t off = 0;
  template <typename V>
  V* take(size_t values) {
    V* p = reinterpret_cast<V*>(base + off);
    off += align256(sizeof(V) * values);
    return p;
  }
};

void scan(const DecayArgs& a, const DecaySegments& sg, const float* G, float* S, const float* init, float* end,
          bool back, hipStream_t st, const Timer& timed) {
  const Scan s = {G, S, init, end, sg.count, a.D, a.DV, back};
  timed("k_decay_scan", st,
        [&] { hipLaunchKernelGGL(k_decay_scan, dim3(a.B * a.Hv * (kTile2 / kThr)), dim3(kThr), 0, st, s); });
}

// Heads of a state that one block of the forward takes: all, unless that leaves CUs without a block. The block's work on
// the state is done for each part of the heads again.
int heads_each(const DecayArgs& a, const DecaySegments& sg) {
  const int rep = a.H / a.Hv, blocks = a.B * a.Hv * sg.count, parts = std::clamp(1024 / blocks, 1, rep);
  return (rep + parts - 1) / parts;
}
// Segments so that `blocks` blocks have one each, those that the GPU holds at once: four a CU in the forward, two in the
// backward. Forward with 512, 1024 and 2048 blocks: 106, 92 and 94 us for 32768 tokens, 202, 201 and 211 for training over
// 4 x 4096; backward with 256, 512 and 1024: 257, 201 and 200.
DecaySegments segments(int U, int NC, int blocks) {
  const int count = std::clamp(blocks / U, 1, NC), len = (NC + count - 1) / count;
  return {(NC + len - 1) / len, len};
}
DecaySegments forward_segments(int U, int NC) { return segments(U, NC, 1024); }
DecaySegments backward_segments(int U, int NC) { return segments(U, NC, 512); }
}  // namespace

DecaySaved decay_saved_view(void* base, int U, int NC, bool keep) {
  DecaySaved s;
  Room r{static_cast<char*>(base)};
  const DecaySegments sg = forward_segments(U, NC);
  const size_t segs = sg.count > 1 ? (size_t)U * sg.count : 0;
  s.S = keep ? r.take<float>((size_t)U * NC * kTile2) : nullptr;
  // needed by the forward alone: after what the backward reads
  s.G = r.take<float>(2 * segs + 1);
  s.D = r.take<float>(segs * kTile2);
  s.bytes = r.off;
  return s;
}

DecayWork decay_work_view(void* base, const DecayArgs& a) {
  DecayWork w;
  Room r{static_cast<char*>(base)};
  const int U = a.B * a.Hv;
  const DecaySegments sg = backward_segments(U, a.NC);
  const size_t segs = sg.count > 1 ? (size_t)U * sg.count : 0;
  w.G = r.take<float>(2 * segs + 1);
  w.dS = r.take<float>(segs * kTile2);
  w.dqh = a.H != a.Hq ? r.take<float>((size_t)a.B * a.H * a.N * a.D) : nullptr;
  w.dkh = a.Hv != a.Hk ? r.take<float>((size_t)a.B * a.Hv * a.N * a.D) : nullptr;
  w.sum = a.per_head ? r.take<double>((size_t)U * a.NC) : nullptr;
  w.bytes = r.off;
  return w;
}

template <typename T>
void launch_decay_forward(const DecayArgs& a, const float* state, void* out, float* final_state, void* saved, bool keep,
                          hipStream_t st, const Timer& timed) {
  const int U = a.B * a.Hv, rep = a.H / a.Hv;
  const DecaySegments sg = forward_segments(U, a.NC);
  const DecaySaved s = decay_saved_view(saved, U, a.NC, keep);
  From from = {state, a.D, a.DV};
  if (sg.count > 1) {
    timed("k_decay_sum", st, [&] {
      hipLaunchKernelGGL((k_decay_sum<T, false>), dim3(U * sg.count), dim3(kThr), 0, st, a, sg, nullptr, s.G, s.D);
    });
    scan(a, sg, s.G, s.D, state, final_state, false, st, timed);
    from = {s.D, 64, 64};
  }
  const auto kernel = sg.count > 1 && !keep && kPartsOf<T> < 3 ? k_decay_out<T, 2> : k_decay_out<T, 3>;
  const int each = heads_each(a, sg);
  timed("k_decay_out", st, [&] {
    hipLaunchKernelGGL(kernel, dim3(U * sg.count * ((rep + each - 1) / each)), dim3(kThr), 0, st, a, sg, each, from,
                       static_cast<T*>(out), sg.count > 1 ? nullptr : final_state, s.S);
  });
}

template <typename T>
void launch_decay_backward(const DecayArgs& a, const void* saved, const void* dout, const float* dfinal, void* dq,
                           void* dk, void* dv, float* dg, float* dstate, void* work, hipStream_t st,
                           const Timer& timed) {
  const int U = a.B * a.Hv;
  const DecaySegments sg = backward_segments(U, a.NC);
  const DecaySaved s = decay_saved_view(const_cast<void*>(saved), U, a.NC, true);
  const DecayWork w = decay_work_view(work, a);
  const T* od = static_cast<const T*>(dout);
  From from = {dfinal, a.D, a.DV};
  if (sg.count > 1) {
    timed("k_decay_sum_back", st, [&] {
      hipLaunchKernelGGL((k_decay_sum<T, true>), dim3(U * sg.count), dim3(kThr), 0, st, a, sg, od, w.G, w.dS);
    });
    scan(a, sg, w.G, w.dS, dfinal, dstate, true, st, timed);
    from = {w.dS, 64, 64};
  }
  timed("k_decay_bwd", st, [&] {
    hipLaunchKernelGGL(k_decay_bwd<T>, dim3(U * sg.count), dim3(kThr), 0, st, a, sg, from, od, s.S,
                       static_cast<T*>(dq), w.dqh, static_cast<T*>(dk), w.dkh, static_cast<T*>(dv), dg, w.sum, dstate);
  });
  if (w.sum)
    timed("k_decay_gate_sum", st, [&] {
      hipLaunchKernelGGL(k_decay_gate_sum, dim3(a.Hv), dim3(kThr), 0, st, w.sum, a.B, a.Hv, a.NC, dg);
    });
  if (w.dqh) launch_sum_heads(w.dqh, static_cast<T*>(dq), a.B, a.Hq, a.H / a.Hq, (int64_t)a.N * a.D, st, timed);
  if (w.dkh) launch_sum_heads(w.dkh, static_cast<T*>(dk), a.B, a.Hk, a.Hv / a.Hk, (int64_t)a.N * a.D, st, timed);
}

#define OAL_DECAY(T)                                                                                               \
  template void launch_decay_forward<T>(const DecayArgs&, const float*, void*, float*, void*, bool, hipStream_t,   \
                                        const Timer&);                                                            \
  template void launch_decay_backward<T>(const DecayArgs&, const void*, const void*, const float*, void*, void*,   \
                                         void*, float*, float*, void*, hipStream_t, const Timer&);
OAL_DECAY(float)
OAL_DECAY(uint16_t)
OAL_DECAY(_Float16)
#undef OAL_DECAY

void launch_decay_step(int kind, const DecayStepArgs& a, hipStream_t st, const Timer& timed) {
  timed("k_decay_step", st, [&] {
    const dim3 grid(a.B * a.Hv), block(kThr);
    if (kind == 0)
      hipLaunchKernelGGL(k_decay_step<float>, grid, block, 0, st, a);
    else if (kind == 1)
      hipLaunchKernelGGL(k_decay_step<uint16_t>, grid, block, 0, st, a);
    else
      hipLaunchKernelGGL(k_decay_step<_Float16>, grid, block, 0, st, a);
  });
}

}  // namespace oal
