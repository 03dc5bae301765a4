// Gated delta rule for gfx950: chunked forward and backward over whole sequences, and
// the recurrence over single tokens.
//
//   S_t = a_t S_{t-1} + k_t u_t^T,  a_t = exp(g_t),  u_t = beta_t z_t,
//   z_t = v_t - a_t S_{t-1}^T k_t,  o_t = scale S_t^T q_t
//
// In chunks of 64 tokens, G the sums of g inside the chunk, S the state before it:
//   A_ij = exp(G_i - G_j) k_i.k_j (j < i),  T = (I + A diag(beta))^-1
//   Z = T (V - e^G K S),  U = beta Z,  S' = e^(G_63) S + K^T (e^(G_63 - G) U)
//   O = scale (e^G Q S + (exp(G_i - G_j) q_i.k_j)_(j <= i) U)
// A chunk maps the state before it to M S + D, with M and D of its own tokens alone:
// T, M and D are formed chunk by chunk at once, then S in a walk of one product per
// chunk, then Z and O chunk by chunk at once. What makes the state is exact to fp32
// whatever the tensors' type (oal_tile.hpp): a state is a sum over all tokens before it and is
// handed on in fp32. T, M, D, S and Z pass through memory in fp32, 16 KB each per 64
// tokens where q, k, v and out are 8 KB: they are what the chunked kernels move most of.
//
// Figures at the kernels: bfloat16, 4 x 4096 tokens of 14 heads and states (3584 chunks),
// with the bytes that the kernel itself reads and writes; a copy reaches 5.2 TB/s.
//
// Decays enter as differences of sums, held in two floats (48 bits): a token that
// forgets nearly everything leaves large sums whose differences still matter.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "oal_common.hpp"
#include "oal_delta.hpp"
#include "oal_tile.hpp"

namespace oal {

namespace {

constexpr int kThr = 256;
constexpr int kTile2 = 64 * 64;
// Smallest log-decay: exp of it is zero, and 64 of them leave the sums' differences exact.
constexpr double kLeast = -1e4;

// Of a chunk's tokens: log2 of the decay up to and with the token, in two parts; beta; the decay since
// the chunk's start and until its end. Formed once, by k_delta_chunk.
struct alignas(16) Gates {
  float hi[64], lo[64], beta[64], since[64], until[64];
};
constexpr int kGates = sizeof(Gates) / sizeof(float);

__device__ __forceinline__ f32x4 four(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
// Decays from token (hi, lo) to tokens r .. r + 3, and from those to it.
__device__ __forceinline__ f32x4 decay_to(const Gates& s, int r, float hi, float lo) {
  const f32x4 h = four(s.hi + r), l = four(s.lo + r);
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_exp2f((h[i] - hi) + (l[i] - lo));
  return y;
}
__device__ __forceinline__ f32x4 decay_from(const Gates& s, int r, float hi, float lo) {
  const f32x4 h = four(s.hi + r), l = four(s.lo + r);
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_exp2f((hi - h[i]) + (lo - l[i]));
  return y;
}
__device__ __forceinline__ void fetch_gates(Gates& s, const float* __restrict__ src, int t) {
  if (t < kGates / 4) reinterpret_cast<float4*>(&s)[t] = reinterpret_cast<const float4*>(src)[t];
}

template <typename T>
__device__ __forceinline__ float beta_at(const DeltaArgs& a, int b, int h, int tok) {
  const int64_t at = b * a.beta.b + h * a.beta.h + tok * a.beta.n;
  return a.beta32 ? static_cast<const float*>(a.beta.p)[at] : get(static_cast<const T*>(a.beta.p) + at);
}

// The first wave of the block; tokens past N decay nothing and write nothing.
template <typename T>
__device__ __forceinline__ void form_gates(Gates& s, const DeltaArgs& a, int b, int h, int tok0, int t) {
  if (t >= 64) return;
  const int tok = tok0 + t;
  double x = 0;
  float beta = 0;
  if (tok < a.N) {
    x = static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + tok * a.g.n];
    x = (x < kLeast ? kLeast : x) * 1.4426950408889634;
    beta = beta_at<T>(a, b, h, tok);
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __shfl_up(x, off, 64);
    if (t >= off) x += y;
  }
  const double end = __shfl(x, 63, 64);
  const float hi = (float)x, lo = (float)(x - (double)hi);
  s.hi[t] = hi;
  s.lo[t] = lo;
  s.beta[t] = beta;
  s.since[t] = __builtin_amdgcn_exp2f(hi + lo);
  s.until[t] = __builtin_amdgcn_exp2f((float)(end - x));
}

template <typename T>
__device__ __forceinline__ const T* rows_of(const Strided& s, int b, int h, int tok0) {
  return static_cast<const T*>(s.p) + b * s.b + h * s.h + (int64_t)tok0 * s.n;
}

// One wave: c[16][16] += a[16][K] b[K][16] of fp32 tiles in LDS (rows of 68) on the fp32 matrix cores.
constexpr int kRow32 = 68;
template <int K>
__device__ __forceinline__ f32x4 mma_f32(const float* a, const float* b, f32x4 c, int lane) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int s = 0; s < K; s += 4)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r * kRow32 + s + g], b[(s + g) * kRow32 + r], c, 0, 0, 0);
  return c;
}

}  // namespace

// Two 64 x 64 products' results in C layout go to LDS rows as bf16 parts.
template <int NP>
__device__ __forceinline__ void put_parts(Tile<NP>& s, int row, int col, float x) {
#pragma unroll
  for (int e = 0; e < NP; ++e) {
    const __bf16 y = static_cast<__bf16>(x);
    s.x[e * kTileElems + tile_at(row, col)] = y;
    x -= static_cast<float>(y);
  }
}

// One chunk by itself: T, and the chunk's map of the state S' = M S + D,
//   M = e^(G_63) - (e^(G_63 - G) beta K)^T T e^G K,  D = (e^(G_63 - G) beta K)^T T V.
// T's diagonal blocks of 16 rows by substitution (a lane per column), then twice
// the rule for two blocks, [L11 0; L21 L22]^-1 = [T11 0; -T22 L21 T11, T22], on the
// fp32 matrix cores. In the products a wave owns 16 columns of M and of D, V's tile in
// the LDS that the triangle leaves: three blocks per CU (53 KB). 68 us, 240 MB: 3.5 TB/s, a
// third of the time the inverse, whose steps wait for each other.
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_chunk(DeltaArgs a, float* __restrict__ Gout, float* __restrict__ Tout,
                                                      float* __restrict__ Mout, float* __restrict__ Dout) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K;
  __shared__ Gates gate;
  // V takes the triangle's place when that is in parts: three blocks of bf16 rows fit a CU
  constexpr int kRoomS = 64 * kRow32 * 4;
  __shared__ alignas(16) char roomS[sizeof(Tile<NP>) > kRoomS ? sizeof(Tile<NP>) : kRoomS];
  float* const S = reinterpret_cast<float*>(roomS);
  Tile<NP>& V = *reinterpret_cast<Tile<NP>*>(roomS);
  struct Solve {
    float L[64 * kRow32], Y[32 * kRow32];
  };
  __shared__ alignas(16) char room[sizeof(Tile<3>) > sizeof(Solve) ? sizeof(Tile<3>) : sizeof(Solve)];
  float* const L = reinterpret_cast<Solve*>(room)->L;
  float* const Y = reinterpret_cast<Solve*>(room)->Y;
  Tile<3>& P = *reinterpret_cast<Tile<3>*>(room);
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0);
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  Incoming<NP, T> ki, vi;
  ki.fetch(rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
  vi.fetch(rows_of<T>(a.v, b, h, tok0), a.v.n, a.DV, live, t);
  form_gates<T>(gate, a, b, h, tok0, t);
  ki.store(K, t);
  lds_sync();
  float* gates = Gout + ((size_t)u * a.NC + ch) * kGates;
  fetch_gates(*reinterpret_cast<Gates*>(gates), reinterpret_cast<const float*>(&gate), t);
  {
    const Frag<NP> k0 = row_frag(K, 16 * w, 0, lane), k1 = row_frag(K, 16 * w, 1, lane);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = 16 * n + c, row = 16 * w + 4 * g;
      f32x4 kk = {};
      if (n <= w) {
        kk = mma(k0, row_frag(K, 16 * n, 0, lane), kk);
        kk = mma(k1, row_frag(K, 16 * n, 1, lane), kk) * decay_to(gate, row, gate.hi[j], gate.lo[j]) * gate.beta[j];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        L[(row + r) * kRow32 + j] = j < row + r ? kk[r] : 0.f;
        S[(row + r) * kRow32 + j] = 0.f;
      }
    }
  }
  lds_sync();
  if (lane < 16) {
    const float* l = L + (16 * w) * kRow32 + 16 * w;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) acc -= l[i * kRow32 + j] * x[j];
      x[i] = acc;
      S[(16 * w + i) * kRow32 + 16 * w + c] = acc;
    }
  }
  lds_sync();
  f32x4 y = {};
  if (w < 2) {
    const int o = 32 * w;
    y = mma_f32<16>(L + (o + 16) * kRow32 + o, S + o * kRow32 + o, y, lane);
#pragma unroll
    for (int r = 0; r < 4; ++r) Y[(16 * w + 4 * g + r) * kRow32 + c] = y[r];
  }
  lds_sync();
  if (w < 2) {
    const int o = 32 * w;
    y = mma_f32<16>(S + (o + 16) * kRow32 + o + 16, Y + 16 * w * kRow32, f32x4{}, lane);
#pragma unroll
    for (int r = 0; r < 4; ++r) S[(o + 16 + 4 * g + r) * kRow32 + o + c] = -y[r];
  }
  lds_sync();
  const int m2 = 16 * (w >> 1), n2 = 16 * (w & 1);
  y = mma_f32<32>(L + (32 + m2) * kRow32, S + n2, f32x4{}, lane);
#pragma unroll
  for (int r = 0; r < 4; ++r) Y[(m2 + 4 * g + r) * kRow32 + n2 + c] = y[r];
  lds_sync();
  y = mma_f32<32>(S + (32 + m2) * kRow32 + 32, Y + n2, f32x4{}, lane);
#pragma unroll
  for (int r = 0; r < 4; ++r) S[(32 + m2 + 4 * g + r) * kRow32 + n2 + c] = -y[r];
  lds_sync();
  // twice: T's columns scaled by e^G times K, T times V; then what the chunk writes of it
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int i = t + kThr * x, r = i >> 3, col = 8 * (i & 7);
      float v[8];
      load_row8(v, S + r * kRow32 + col);
      if (side == 0) {
        float4* dst = reinterpret_cast<float4*>(Tout + at + 8 * i);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        const f32x4 g0 = four(gate.since + col), g1 = four(gate.since + col + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= e < 4 ? g0[e] : g1[e - 4];
      }
      const Frag<3> f = split<3>(v);
#pragma unroll
      for (int e = 0; e < 3; ++e) *reinterpret_cast<bf16x8*>(P.x + e * kTileElems + tile_at(r, col)) = f.p[e];
    }
    lds_sync();
    if (side == 1) {
      vi.store(V, t);
      lds_sync();
    }
    const Tile<NP>& B = side == 0 ? K : V;
    const Frag<NP> b0 = col_frag(B, 16 * w, 0, lane), b1 = col_frag(B, 16 * w, 1, lane);
    f32x4 z[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      z[m] = mma(row_frag(P, 16 * m, 0, lane), b0, f32x4{});
      if (m >= 2) z[m] = mma(row_frag(P, 16 * m, 1, lane), b1, z[m]);
      const f32x4 x = four(gate.beta + 16 * m + 4 * g) * four(gate.until + 16 * m + 4 * g);
      z[m] *= side == 0 ? -x : x;
    }
    const Frag<3> z0 = acc_frag<3>(z[0], z[1]), z1 = acc_frag<3>(z[2], z[3]);
    const float last = gate.since[63];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 x = mma(col_frag_perm(K, 16 * m, 0, lane), z0, f32x4{});
      x = mma(col_frag_perm(K, 16 * m, 1, lane), z1, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * m + 4 * g + i, col = 16 * w + c;
        (side == 0 ? Mout : Dout)[at + row * 64 + col] = side == 0 && row == col ? x[i] + last : x[i];
      }
    }
    lds_sync();
  }
}

// A walk over maps of 64 x 64 states, S -> M S + D, or back through them, S -> M^T S + D
// (M's transpose where TR): a block per chain and 16 columns, a wave per 16 rows, who
// hand each other their rows through LDS once per map. What a map needs of memory is
// loaded kAhead maps before. On the fp32 matrix cores, whose operands are M and S as
// they lie in registers and LDS (sum index 16 q + 4 g + e of instruction q, e): their
// 16 instructions per map are slower than 12 of bf16 parts, but there is nothing to split.
// 58 us for 64 maps, 0.9 us each: bound by the way of a state through LDS, 16
// instructions and their sum, not by the 176 MB that it moves meanwhile (3.0 TB/s).
struct Walk {
  const float* M;     // [units][maps][64][64]
  const float* D;
  const float* init;  // [rows][cols] state the walk starts from, by unit (segs == 1) or segment (null: zero)
  float* each;        // [units][maps][64][64]: the state before each map (without MAPS)
  float* end;         // the same: the state after the last map (null: not wanted)
  float* mend;        // with MAPS: the product of the segment's maps
  int maps, segs, len, units, rows, cols;
  bool back;
};

constexpr int kAhead = 4;

// With MAPS the block walks the same columns of the maps' product beside its own (from the
// unit matrix, nothing added): twice the products from one load of the maps.
template <bool TR, bool MAPS>
__global__ __launch_bounds__(kThr) void k_delta_walk(Walk a) {
  constexpr int SETS = MAPS ? 2 : 1;
  __shared__ f32x4 rows[2][SETS][4][64];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  // a chain's column groups on one XCD (blocks go round the 8 of them): they share its maps
  const int chains = a.units * a.segs, id = blockIdx.x, whole = chains / 8 * 32;
  const int chain = id < whole ? id % 8 + id / 32 * 8 : chains / 8 * 8 + (id - whole) / 4;
  const int group = id < whole ? id / 8 % 4 : (id - whole) % 4;
  const int u = chain / a.segs, seg = chain % a.segs;
  const int first = seg * a.len, count = min(a.len, a.maps - first);
  const int col = 16 * group + c, row = 16 * w + 4 * g;
  const size_t base = ((size_t)u * a.maps + first) * kTile2;
  auto slot = [&](int i) { return ((size_t)chain * a.rows + row + i) * a.cols + col; };
  auto held = [&](int i) { return row + i < a.rows && col < a.cols; };
  float m[kAhead][16], d[kAhead][4];
  auto fetch = [&](int n, float (&mm)[16], float (&dd)[4]) {
    n = min(n, count - 1);
    const size_t at = base + (size_t)(a.back ? count - 1 - n : n) * kTile2;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = 16 * q + 4 * g;
      if constexpr (TR) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mm[4 * q + e] = a.M[at + (k + e) * 64 + 16 * w + c];
      } else {
        const float4 v = *reinterpret_cast<const float4*>(a.M + at + (16 * w + c) * 64 + k);
        mm[4 * q] = v.x, mm[4 * q + 1] = v.y, mm[4 * q + 2] = v.z, mm[4 * q + 3] = v.w;
      }
      dd[q] = a.D[at + (row + q) * 64 + col];
    }
  };
  f32x4 S[SETS];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    S[0][i] = a.init && held(i) ? a.init[slot(i)] : 0.f;
    if constexpr (MAPS) S[1][i] = row + i == col ? 1.f : 0.f;
  }
  asm volatile("" : "+v"(S[0]));  // here, not in the walk, is waited for it
#pragma unroll
  for (int n = 0; n < kAhead; ++n) fetch(n, m[n], d[n]);
  // the number of loads in flight is the same on every way to a step, so that it waits for its own
  auto step = [&](int n, int x) {
#pragma unroll
    for (int p = 0; p < SETS; ++p) rows[x & 1][p][w][lane] = S[p];
    if constexpr (!MAPS) {
      const size_t at = base + (size_t)(a.back ? count - 1 - n : n) * kTile2;
#pragma unroll
      for (int i = 0; i < 4; ++i) a.each[at + (row + i) * 64 + col] = S[0][i];
    }
    f32x4 next[SETS][4] = {{{d[x][0], d[x][1], d[x][2], d[x][3]}}};
    lds_sync();
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int p = 0; p < SETS; ++p) {
        const f32x4 v = rows[x & 1][p][q][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          next[p][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[x][4 * q + e], v[e], next[p][q], 0, 0, 0);
      }
#pragma unroll
    for (int p = 0; p < SETS; ++p) S[p] = (next[p][0] + next[p][1]) + (next[p][2] + next[p][3]);
    // behind the products, into the registers that they are done with: loaded before, the
    // values would go through others and be waited for at once
    __builtin_amdgcn_sched_barrier(0);
    fetch(n + kAhead, m[x], d[x]);
  };
  int n = 0;
  for (; n + kAhead <= count; n += kAhead)
#pragma unroll
    for (int x = 0; x < kAhead; ++x) step(n + x, x);
#pragma unroll
  for (int x = 0; x < kAhead - 1; ++x)
    if (n + x < count) step(n + x, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!held(i)) continue;
    if (a.end) a.end[slot(i)] = S[0][i];
    if constexpr (MAPS) a.mend[slot(i)] = S[1][i];
  }
}

// The outputs of one chunk for `each` output heads of a state head. First Z = T (V -
// e^G K S), a wave per 16 columns, to LDS as U = beta Z; then per output head, transposed: a
// wave's 16 queries are the columns, so the scores are an operand of the product
// with U as they are. What goes on to the backward (KEEP) is exact to fp32; the outputs take
// two parts per value for 16-bit tensors, twice their precision: one rounding is the output's own.
// 80 us, 294 MB: 3.7 TB/s, with three blocks per CU (42 KB of LDS) where nothing is kept.
template <typename T, bool KEEP>
__global__ __launch_bounds__(kThr) void k_delta_out(DeltaArgs a, int each, const float* __restrict__ Gin,
                                                    const float* __restrict__ Tin, const float* __restrict__ Sin,
                                                    float* __restrict__ Zout, T* __restrict__ out) {
  constexpr int NP = kPartsOf<T>, NZ = KEEP || NP == 3 ? 3 : 2, NO = NP == 3 ? 3 : 2;
  __shared__ Tile<NP> K;
  __shared__ Tile<NZ> S, U;
  __shared__ Gates gate;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int rep = a.H / a.Hv, parts = (rep + each - 1) / each;
  const int part = blockIdx.x % parts, ch = blockIdx.x / parts % a.NC, u = blockIdx.x / parts / a.NC;
  const int b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  Incoming<NP, T> ki;
  Incoming<NZ, float> si, ti;
  ki.fetch(rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
  si.fetch(Sin + at, 64, 64, 64, t);
  ti.fetch(Tin + at, 64, 64, 64, t);
  const T* v = rows_of<T>(a.v, b, h, tok0) + min(own, a.DV - 1);
  f32x4 z[4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * m + 4 * g + i;
      z[m][i] = get(v + min(row, live - 1) * a.v.n);
      z[m][i] = row < live && own < a.DV ? z[m][i] : 0.f;
    }
  fetch_gates(gate, Gin + at / kTile2 * kGates, t);
  ki.store(K, t);
  si.store(S, t);
  ti.store(U, t);
  lds_sync();
  {
    const Frag<NZ> s0 = col_frag(S, 16 * w, 0, lane), s1 = col_frag(S, 16 * w, 1, lane);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 x = mma(row_frag(K, 16 * m, 0, lane), s0, f32x4{});
      x = mma(row_frag(K, 16 * m, 1, lane), s1, x);
      z[m] -= four(gate.since + 16 * m + 4 * g) * x;
    }
  }
  {
    const Frag<NZ> r0 = acc_frag<NZ>(z[0], z[1]), r1 = acc_frag<NZ>(z[2], z[3]);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      z[m] = mma(row_frag_perm(U, 16 * m, 0, lane), r0, f32x4{});
      if (m >= 2) z[m] = mma(row_frag_perm(U, 16 * m, 1, lane), r1, z[m]);
    }
  }
  lds_sync();
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const f32x4 u4 = four(gate.beta + 16 * m + 4 * g) * z[m];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * m + 4 * g + i;
      if (KEEP && part == 0) Zout[at + row * 64 + own] = z[m][i];
      put_parts(U, row, own, u4[i]);
    }
  }
  lds_sync();
  const float since = a.scale * gate.since[own], hi = gate.hi[own], lo = gate.lo[own];
  for (int o = h * rep + part * each; o < min(h * rep + (part + 1) * each, (h + 1) * rep); ++o) {
    const T* q = rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0) + own * a.q.n;
    Frag<NP> qf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) qf[s] = global_frag<NP>(q + 32 * s + 8 * g, own < live && 32 * s + 8 * g < a.D);
    f32x4 acc[4] = {}, p[4] = {};
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int s = 0; s < 2; ++s) acc[m] = mma(col_frag<NO>(S, 16 * m, s, lane), qf[s], acc[m]);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] *= since;
      if (m > w) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) p[m] = mma(row_frag(K, 16 * m, s, lane), qf[s], p[m]);
      const f32x4 y = p[m] * a.scale * decay_from(gate, 16 * m + 4 * g, hi, lo);
#pragma unroll
      for (int i = 0; i < 4; ++i) p[m][i] = 16 * m + 4 * g + i <= own ? y[i] : 0.f;
    }
    const Frag<NO> p0 = acc_frag<NO>(p[0], p[1]), p1 = acc_frag<NO>(p[2], p[3]);
    T* dst = out + (((size_t)b * a.H + o) * a.N + tok0 + own) * a.DV;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      acc[m] = mma(col_frag_perm<NO>(U, 16 * m, 0, lane), p0, acc[m]);
      if (w >= 2) acc[m] = mma(col_frag_perm<NO>(U, 16 * m, 1, lane), p1, acc[m]);
      if (own < live && 16 * m + 4 * g < a.DV) store4(dst + 16 * m + 4 * g, acc[m]);
    }
  }
}

// ---------------------------------------------------------------------------
// Backward. Per chunk at once, from its own outputs: the gradient E of its u and, with
// what it does to the state before through them, F; the walk back over the chunks'
// maps, dS = M^T dS' + F; and from dS', S and Z everything else of the chunk at once:
//   E = D^T dO,  F = scale (e^G Q)^T dO - (e^G K)^T T^T (beta E)
//   dU = E + e^(G_63 - G) K dS',  dZ = dV = T^T (beta dU)
// Decays' gradients are sums of terms that cancel, so all of it is exact to fp32.
// k_delta_bwd_local: 60 us, 264 MB: 4.4 TB/s, three blocks per CU (two: 69 us).
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThr, kPartsOf<T> == 1 ? 3 : 1)
void k_delta_bwd_local(DeltaArgs a, const T* __restrict__ dout,
                                                          const float* __restrict__ Gin, const float* __restrict__ Tin,
                                                          float* __restrict__ E, float* __restrict__ F) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K, Q, O;
  __shared__ Tile<3> P;
  __shared__ Gates gate;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  // the next head's rows are on their way while one is worked on, the solved triangle behind the last
  Incoming<NP, T> ki, qi, oi;
  Incoming<3, float> ti;
  const int each = a.H / a.Hv, o1 = (h + 1) * each;
  auto fetch = [&](int o) {
    qi.fetch(rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0), a.q.n, a.D, live, t);
    oi.fetch(dout + (((size_t)b * a.H + o) * a.N + tok0) * a.DV, a.DV, a.DV, live, t);
  };
  ki.fetch(rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
  fetch(h * each);
  fetch_gates(gate, Gin + at / kTile2 * kGates, t);
  ki.store(K, t);
  f32x4 e[4] = {}, f[4] = {};
  for (int o = h * each; o < o1; ++o) {
    if (o > h * each) lds_sync();
    qi.store(Q, t);
    oi.store(O, t);
    lds_sync();
    if (o + 1 < o1)
      fetch(o + 1);
    else
      ti.fetch(Tin + at, 64, 64, 64, t);
    // the scores, queries by keys = own: to LDS with the queries along a row
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 p = {};
      if (m >= w)
#pragma unroll
        for (int s = 0; s < 2; ++s) p = mma(row_frag(Q, 16 * m, s, lane), row_frag(K, 16 * w, s, lane), p);
      const f32x4 y = p * a.scale * decay_to(gate, 16 * m + 4 * g, gate.hi[own], gate.lo[own]);
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = own <= 16 * m + 4 * g + i ? y[i] : 0.f;
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        const bf16x4 y = __builtin_bit_cast(bf16x4, pack4(v));
        *reinterpret_cast<bf16x4*>(P.x + x * kTileElems + tile_at(own, 16 * m + 4 * g)) = y;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] -= static_cast<float>(y[i]);
      }
    }
    Frag<NP> of[2];
    Frag<3> og[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      of[s] = col_frag(O, 16 * w, s, lane);
      float v[8];
      const f32x4 g0 = a.scale * four(gate.since + 32 * s + 8 * g);
      const f32x4 g1 = a.scale * four(gate.since + 32 * s + 8 * g + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = 0.f;
#pragma unroll
        for (int x = NP - 1; x >= 0; --x) v[j] += static_cast<float>(of[s].p[x][j]);
        v[j] *= j < 4 ? g0[j] : g1[j - 4];
      }
      og[s] = split<3>(v);
    }
    lds_sync();
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (m < 2) e[m] = mma(row_frag(P, 16 * m, 0, lane), of[0], e[m]);
      e[m] = mma(row_frag(P, 16 * m, 1, lane), of[1], e[m]);
#pragma unroll
      for (int s = 0; s < 2; ++s) f[m] = mma(col_frag(Q, 16 * m, s, lane), og[s], f[m]);
    }
  }
  lds_sync();
  ti.store(P, t);
  f32x4 z[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) E[at + (16 * m + 4 * g + i) * 64 + own] = e[m][i];
    e[m] *= four(gate.beta + 16 * m + 4 * g);
  }
  const Frag<3> e0 = acc_frag<3>(e[0], e[1]), e1 = acc_frag<3>(e[2], e[3]);
  lds_sync();
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    z[m] = mma(col_frag_perm(P, 16 * m, 1, lane), e1, f32x4{});
    if (m < 2) z[m] = mma(col_frag_perm(P, 16 * m, 0, lane), e0, z[m]);
    z[m] *= -four(gate.since + 16 * m + 4 * g);
  }
  const Frag<3> z0 = acc_frag<3>(z[0], z[1]), z1 = acc_frag<3>(z[2], z[3]);
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    f[m] = mma(col_frag_perm(K, 16 * m, 0, lane), z0, f[m]);
    f[m] = mma(col_frag_perm(K, 16 * m, 1, lane), z1, f[m]);
#pragma unroll
    for (int i = 0; i < 4; ++i) F[at + (16 * m + 4 * g + i) * 64 + own] = f[m][i];
  }
}

// Row `own` of a 64 x 64 fp32 tile as an operand, and as the accumulators' four-value pieces.
__device__ __forceinline__ void own_row(Frag<3> (&f)[2], const float* row, int g) {
#pragma unroll
  for (int s = 0; s < 2; ++s) f[s] = global_frag<3>(row + 32 * s + 8 * g, true);
}

// Everything of one chunk and state head that the walk back leaves: with M_ij =
// -beta_j exp(G_i - G_j) dZ_i.Z_j (j < i), D_ij = scale exp(G_i - G_j) dO_i.U_j (j <= i),
//   dq = scale e^G dO S^T + D K               (per output head)
//   dk = M K - e^G dZ S^T                     (k as what reads the state)
//      + M^T K + D^T Q + e^(G_63 - G) U dS'^T (k as what writes it)
//   dbeta_j = dU_j.Z_j - sum_(i > j) A_ij dZ_i.Z_j
//   dG_i = the products' terms with e^(G_i) less those with e^(-G_i)
//        = sum_j (D_ij q_i.k_j + M_ij k_i.k_j) - sum_j (D_ji q_j.k_i + M_ji k_j.k_i)  (j != i)
//          + scale e^(G_i) q_i.(S dO_i) - e^(G_i) k_i.(S dZ_i) - e^(G_63 - G_i) k_i.(dS' U_i),
//        and at the chunk's end e^(G_63) <S, dS'> + sum_j e^(G_63 - G_j) k_j.(dS' U_j);
// dg the sums of dG from each token to the chunk's end. Terms that do not decay (j = i,
// the last token's write) are left out rather than cancelled: where all decay is
// strong, dg is far smaller than they are. All products are transposed: a wave's 16
// tokens are the columns. What goes into dq and dk alone is cut to two bf16 parts
// (16 bits) for 16-bit tensors, which then round once themselves; dg and dbeta see three.
// 205 us, 470 MB: 2.3 TB/s. Two blocks per CU (76 KB of LDS, 251 registers) do not
// cover its loads and its 13 products of 64 x 64 x 64 in 3 to 6 instructions each.
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_bwd_out(DeltaArgs a, const T* __restrict__ dout,
                                                        const float* __restrict__ Gin, const float* __restrict__ Tin,
                                                        const float* __restrict__ Sin, const float* __restrict__ Zin,
                                                        const float* __restrict__ E,
                                                        const float* __restrict__ dSin, T* __restrict__ dq,
                                                        float* __restrict__ dqh, T* __restrict__ dk,
                                                        float* __restrict__ dkh, T* __restrict__ dv,
                                                        float* __restrict__ dg, void* __restrict__ dbeta) {
  // what goes into dq and dk alone takes two parts for 16-bit tensors
  constexpr int NP = kPartsOf<T>, NO = NP == 3 ? 3 : 2;
  __shared__ Tile<NP> K, Q, O;
  __shared__ Tile<3> Z, X;
  __shared__ Gates gate;
  __shared__ float dG[64], part[4], dotU[4][64];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  const T* krows = rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0);
  Incoming<NP, T> ki;
  Incoming<3, float> xi, zi;
  ki.fetch(krows, a.k.n, a.D, live, t);
  xi.fetch(dSin + at, 64, 64, 64, t);
  zi.fetch(Tin + at, 64, 64, 64, t);
  Frag<3> zf[2], dzf[2];
  own_row(zf, Zin + at + own * 64, g);
  f32x4 e[4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) e[m][i] = E[at + (16 * m + 4 * g + i) * 64 + own];
  // <S, dS'>
  float ends = 0.f;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = 4 * (t + kThr * x);
    const f32x4 s = load4(Sin + at + i), d = load4(dSin + at + i);
    ends += s[0] * d[0] + s[1] * d[1] + s[2] * d[2] + s[3] * d[3];
  }
  fetch_gates(gate, Gin + at / kTile2 * kGates, t);
  ki.store(K, t);
  xi.store(X, t);
  zi.store(Z, t);
  lds_sync();
  zi.fetch(Zin + at, 64, 64, 64, t);
  ends *= gate.since[63];
  const float beta = gate.beta[own], hi = gate.hi[own], lo = gate.lo[own];
  f32x4 reads[4] = {}, writes[4] = {};
  float dot = 0.f;    // of dbeta
  float decay = 0.f;  // of dG
  f32x4 kv[4];
  {
    const float until = beta * gate.until[own];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      kv[n] = f32x4{};
      if (own < live && 16 * n + 4 * g < a.D) kv[n] = load4(krows + own * a.k.n + 16 * n + 4 * g);
      f32x4 x = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) x = mma(row_frag(X, 16 * n, s, lane), zf[s], x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = until * x[i];
        writes[n][i] += y;
        // what the last token writes does not decay
        const float z = own < live - 1 ? kv[n][i] * y : 0.f;
        ends += z;
        decay -= z;
      }
    }
  }
  ends = wave_sum(ends);
  if (lane == 0) part[w] = ends;
  {
    // dU and dZ, columns of the values: own
    const Frag<3> s0 = col_frag(X, 16 * w, 0, lane), s1 = col_frag(X, 16 * w, 1, lane);
    float dots[16];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 x = mma(row_frag(K, 16 * m, 0, lane), s0, f32x4{});
      x = mma(row_frag(K, 16 * m, 1, lane), s1, x);
      e[m] += four(gate.until + 16 * m + 4 * g) * x;
#pragma unroll
      for (int i = 0; i < 4; ++i) dots[4 * m + i] = e[m][i] * Zin[at + (16 * m + 4 * g + i) * 64 + own];
      e[m] *= four(gate.beta + 16 * m + 4 * g);
    }
    // sums over the 16 lanes of a row group; lane c ends with row 16 (c / 4) + 4 g + c % 4
#pragma unroll
    for (int half = 8; half > 0; half >>= 1)
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const bool up = c & half;
        const float mine = up ? dots[i + half] : dots[i], other = up ? dots[i] : dots[i + half];
        dots[i] = mine + __shfl_xor(other, half, 64);
      }
    dotU[w][16 * (c >> 2) + 4 * g + (c & 3)] = dots[0];
    const Frag<3> e0 = acc_frag<3>(e[0], e[1]), e1 = acc_frag<3>(e[2], e[3]);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      e[m] = mma(col_frag_perm(Z, 16 * m, 1, lane), e1, f32x4{});
      if (m < 2) e[m] = mma(col_frag_perm(Z, 16 * m, 0, lane), e0, e[m]);
    }
  }
  lds_sync();
  zi.store(Z, t);
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * m + 4 * g + i;
      put_parts(X, row, own, e[m][i]);
      if (row < live && own < a.DV) put(dv + ((size_t)u * a.N + tok0 + row) * a.DV + own, e[m][i]);
    }
  lds_sync();
#pragma unroll
  for (int s = 0; s < 2; ++s) dzf[s] = row_frag(X, 16 * w, s, lane);
  {
    // M^T: rows j, columns i = own
    f32x4 m[4] = {};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n > w) continue;
      f32x4 kk = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        m[n] = mma(row_frag(Z, 16 * n, s, lane), dzf[s], m[n]);
        kk = mma(row_frag(K, 16 * n, s, lane), row_frag(K, 16 * w, s, lane), kk);
      }
      const f32x4 y = -four(gate.beta + 16 * n + 4 * g) * decay_from(gate, 16 * n + 4 * g, hi, lo) * m[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[n][i] = 16 * n + 4 * g + i < own ? y[i] : 0.f;
        decay += m[n][i] * kk[i];
      }
    }
    const Frag<NO> m0 = acc_frag<NO>(m[0], m[1]), m1 = acc_frag<NO>(m[2], m[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      reads[n] = mma(col_frag_perm(K, 16 * n, 0, lane), m0, reads[n]);
      if (w >= 2) reads[n] = mma(col_frag_perm(K, 16 * n, 1, lane), m1, reads[n]);
    }
  }
  xi.fetch(Sin + at, 64, 64, 64, t);
  {
    // M: rows i, columns j = own
    f32x4 m[4] = {};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (n < w) continue;
      f32x4 kk = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        m[n] = mma(row_frag(X, 16 * n, s, lane), zf[s], m[n]);
        kk = mma(row_frag(K, 16 * n, s, lane), row_frag(K, 16 * w, s, lane), kk);
      }
      const f32x4 y = decay_to(gate, 16 * n + 4 * g, hi, lo) * m[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = own < 16 * n + 4 * g + i ? y[i] : 0.f;
        dot -= x * kk[i];
        m[n][i] = -beta * x;
        decay -= m[n][i] * kk[i];
      }
    }
    const Frag<NO> m0 = acc_frag<NO>(m[0], m[1]), m1 = acc_frag<NO>(m[2], m[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (w < 2) writes[n] = mma(col_frag_perm(K, 16 * n, 0, lane), m0, writes[n]);
      writes[n] = mma(col_frag_perm(K, 16 * n, 1, lane), m1, writes[n]);
    }
  }
  dot = group_sum(dot) + ((dotU[0][own] + dotU[1][own]) + (dotU[2][own] + dotU[3][own]));
  if (g == 0 && own < live) {
    const size_t x = (size_t)u * a.N + tok0 + own;
    if (a.beta32)
      static_cast<float*>(dbeta)[x] = dot;
    else
      put(static_cast<T*>(dbeta) + x, dot);
  }
  lds_sync();
  xi.store(X, t);
  const int each = a.H / a.Hv, o1 = (h + 1) * each;
  Incoming<NP, T> qi, oi;
  auto fetch = [&](int o) {
    qi.fetch(rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0), a.q.n, a.D, live, t);
    oi.fetch(dout + (((size_t)b * a.H + o) * a.N + tok0) * a.DV, a.DV, a.DV, live, t);
  };
  fetch(h * each);
  lds_sync();
  const float since = gate.since[own];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    f32x4 x = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) x = mma(row_frag(X, 16 * n, s, lane), dzf[s], x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      reads[n][i] -= since * x[i];
      decay -= kv[n][i] * since * x[i];
    }
  }
  for (int o = h * each; o < o1; ++o) {
    const T* qrows = rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0);
    const size_t orow = ((size_t)b * a.H + o) * a.N + tok0;
    if (o > h * each) lds_sync();
    qi.store(Q, t);
    oi.store(O, t);
    lds_sync();
    if (o + 1 < o1) fetch(o + 1);
    Frag<NP> of[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) of[s] = row_frag(O, 16 * w, s, lane);
    f32x4 acc[4], p[4] = {};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      f32x4 x = {}, qk = {}, qv = {};
      if (own < live && 16 * n + 4 * g < a.D) qv = load4(qrows + own * a.q.n + 16 * n + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s) x = mma(row_frag(X, 16 * n, s, lane), of[s], x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[n][i] = a.scale * since * x[i];
        decay += qv[i] * acc[n][i];
      }
      if (n > w) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        p[n] = mma(row_frag(Z, 16 * n, s, lane), of[s], p[n]);
        qk = mma(row_frag(K, 16 * n, s, lane), row_frag(Q, 16 * w, s, lane), qk);
      }
      const f32x4 y = a.scale * four(gate.beta + 16 * n + 4 * g) * decay_from(gate, 16 * n + 4 * g, hi, lo) * p[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 16 * n + 4 * g + i;
        p[n][i] = j <= own ? y[i] : 0.f;
        decay += j < own ? p[n][i] * qk[i] : 0.f;
      }
    }
    {
      const Frag<NO> p0 = acc_frag<NO>(p[0], p[1]), p1 = acc_frag<NO>(p[2], p[3]);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        acc[n] = mma(col_frag_perm(K, 16 * n, 0, lane), p0, acc[n]);
        if (w >= 2) acc[n] = mma(col_frag_perm(K, 16 * n, 1, lane), p1, acc[n]);
        if (own < live && 16 * n + 4 * g < a.D) {
          if (dqh)
            store4(dqh + (orow + own) * a.D + 16 * n + 4 * g, acc[n]);
          else
            store4(dq + (orow + own) * a.D + 16 * n + 4 * g, acc[n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      p[n] = f32x4{};
      if (n < w) continue;
      f32x4 qk = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        p[n] = mma(row_frag(O, 16 * n, s, lane), zf[s], p[n]);
        qk = mma(row_frag(Q, 16 * n, s, lane), row_frag(K, 16 * w, s, lane), qk);
      }
      const f32x4 y = a.scale * beta * decay_to(gate, 16 * n + 4 * g, hi, lo) * p[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * n + 4 * g + i;
        p[n][i] = own <= row ? y[i] : 0.f;
        decay -= own < row ? p[n][i] * qk[i] : 0.f;
      }
    }
    const Frag<NO> p0 = acc_frag<NO>(p[0], p[1]), p1 = acc_frag<NO>(p[2], p[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (w < 2) writes[n] = mma(col_frag_perm(Q, 16 * n, 0, lane), p0, writes[n]);
      writes[n] = mma(col_frag_perm(Q, 16 * n, 1, lane), p1, writes[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (own < live && 16 * n + 4 * g < a.D) {
      const f32x4 x = reads[n] + writes[n];
      const size_t row = ((size_t)u * a.N + tok0 + own) * a.D + 16 * n + 4 * g;
      if (dkh)
        store4(dkh + row, x);
      else
        store4(dk + row, x);
    }
  }
  decay = group_sum(decay);
  if (g == 0) dG[own] = decay;
  lds_sync();
  if (w == 0) {
    double x = dG[lane];
    if (lane == 63) x += ((double)part[0] + part[1]) + ((double)part[2] + part[3]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double y = __shfl_down(x, off, 64);
      if (lane + off < 64) x += y;
    }
    if (lane < live) dg[(size_t)u * a.N + tok0 + lane] = (float)x;
  }
}

// Gradients of heads that several heads share: their sums, in order. dst
// [B][heads][N][D] of src [B][heads each][N][D].
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_sum_heads(const float* __restrict__ src, T* __restrict__ dst, int each,
                                                          int64_t head, int64_t total) {
  const int64_t x = ((int64_t)blockIdx.x * kThr + threadIdx.x) * 4;
  if (x >= total) return;
  const int64_t bh = x / head, in = x % head;
  f32x4 s = {};
  for (int e = 0; e < each; ++e) s += load4(src + (bh * each + e) * head + in);
  store4(dst + x, s);
}

// ---------------------------------------------------------------------------
// The recurrence itself, for single tokens: a block per state head holds the
// state, 4 x 4 values per thread, for all N tokens and writes it back. Bound by the state,
// once there and back: 256 users of 14 states 29 us, 119 MB at 4.1 TB/s; one user 6.6 us, a
// launch and its latencies.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_step(DeltaStepArgs a) {
  __shared__ float sum[4][64];
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
  // sums over the rows of x[4] per column, all columns c0 .. c0 + 3 of this thread
  auto over_rows = [&](float (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = group_sum(x[j]);
    lds_sync();
    if (lane < 16)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[w][c0 + j] = x[j];
    lds_sync();
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (sum[0][c0 + j] + sum[1][c0 + j]) + (sum[2][c0 + j] + sum[3][c0 + j]);
  };
  for (int n = 0; n < a.N; ++n) {
    const float decay = expf(static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + n * a.g.n]);
    const int64_t bx = b * a.beta.b + h * a.beta.h + n * a.beta.n;
    const float beta = a.beta32 ? static_cast<const float*>(a.beta.p)[bx] : get(static_cast<const T*>(a.beta.p) + bx);
    float kr[4], x[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kr[i] = d0 + i < a.Dk ? get(k + n * a.k.n + d0 + i) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] *= decay;
        x[j] += kr[i] * s[i][j];
      }
    }
    over_rows(x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float vj = c0 + j < a.Dv ? get(v + n * a.v.n + c0 + j) : 0.f;
      const float uj = beta * (vj - x[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i][j] += kr[i] * uj;
    }
    for (int o = h * each; o < (h + 1) * each; ++o) {
      const T* q = static_cast<const T*>(a.q.p) + b * a.q.b + (o / (a.H / a.Hq)) * a.q.h + n * a.q.n;
      float y[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float qi = d0 + i < a.Dk ? get(q + d0 + i) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += qi * s[i][j];
      }
      over_rows(y);
      T* out = static_cast<T*>(a.out) + (((size_t)b * a.H + o) * a.N + n) * a.Dv;
      if (t < 16)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c0 + j < a.Dv) put(out + c0 + j, a.scale * y[j]);
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
  float* take(size_t values) {
    float* p = reinterpret_cast<float*>(base + off);
    off += align256(4 * values);
    return p;
  }
};

// A chunk takes a walk about the same time (0.85 us) whatever happens beside it, so long
// walks of few chains are cut into segments: their maps' products at once (a chunk 1.6
// times as long), a walk over those, then the segments from their own states. In units of a
// chunk's time; two further launches cost about 20, and 512 blocks run at once. 32768
// tokens of 14 states: 9 segments 205 us (4: 218, 18: 213; one walk 430); 1000 tokens of 4:
// one walk 15 us (4 segments 26); 4 x 4096 tokens of 14: one walk 58 us (4 segments 104).
struct Segments {
  int count, len;
};
Segments segments(int U, int NC) {
  auto rounds = [](int64_t blocks) { return (double)((blocks + 511) / 512); };
  Segments best{1, NC};
  double least = NC * rounds(4LL * U);
  for (int len = 4; 2 * len <= NC; ++len) {
    const int n = (NC + len - 1) / len;
    const double cost = 2.6 * len * rounds(4LL * U * n) + n * rounds(4LL * U) + 20;
    if (cost < least) least = cost, best = {n, len};
  }
  return best;
}

template <bool TR>
void walk(const DeltaArgs& g, const float* M, const float* D, const float* init, float* each, float* end,
          float* scratch, bool back, hipStream_t st, const Timer& timed) {
  const int U = g.B * g.Hv, NC = g.NC;
  const Segments sg = segments(U, NC);
  auto launch = [&](const Walk& a, auto tr, auto maps) {
    timed("k_delta_walk", st, [&] {
      hipLaunchKernelGGL((k_delta_walk<decltype(tr)::value, decltype(maps)::value>), dim3(a.units * a.segs * 4),
                         dim3(kThr), 0, st, a);
    });
  };
  using Tr = std::integral_constant<bool, TR>;
  if (sg.count == 1) {
    launch({M, D, init, each, end, nullptr, NC, 1, NC, U, g.D, g.DV, back}, Tr{}, std::false_type{});
    return;
  }
  const size_t part = (size_t)U * sg.count * kTile2;
  float *segM = scratch, *segD = scratch + part, *segS = scratch + 2 * part;
  launch({M, D, nullptr, nullptr, segD, segM, NC, sg.count, sg.len, U, 64, 64, back}, Tr{}, std::true_type{});
  // the products stand as they act, whichever way the walk goes
  launch({segM, segD, init, segS, end, nullptr, sg.count, 1, sg.count, U, g.D, g.DV, back}, std::false_type{},
         std::false_type{});
  launch({M, D, segS, each, nullptr, nullptr, NC, sg.count, sg.len, U, 64, 64, back}, Tr{}, std::false_type{});
}
size_t walk_scratch(int U, int NC) {
  const Segments sg = segments(U, NC);
  return sg.count == 1 ? 0 : (size_t)3 * U * sg.count * kTile2;
}
}  // namespace

DeltaSaved delta_saved_view(void* base, int U, int NC, bool keep) {
  DeltaSaved s;
  Room r{static_cast<char*>(base)};
  const size_t tiles = (size_t)U * NC * kTile2;
  s.G = r.take((size_t)U * NC * kGates);
  s.T = r.take(tiles);
  s.M = r.take(tiles);
  s.S = r.take(tiles);
  s.Z = keep ? r.take(tiles) : nullptr;
  // needed by the forward alone: after what the backward reads
  s.D = r.take(tiles);
  s.scratch = r.take(walk_scratch(U, NC));
  s.bytes = r.off;
  return s;
}

DeltaWork delta_work_view(void* base, const DeltaArgs& a) {
  DeltaWork w;
  Room r{static_cast<char*>(base)};
  const int U = a.B * a.Hv;
  const size_t tiles = (size_t)U * a.NC * kTile2;
  w.E = r.take(tiles);
  w.F = r.take(tiles);
  w.dS = r.take(tiles);
  w.scratch = r.take(walk_scratch(U, a.NC));
  w.dqh = a.H != a.Hq ? r.take((size_t)a.B * a.H * a.N * a.D) : nullptr;
  w.dkh = a.Hv != a.Hk ? r.take((size_t)a.B * a.Hv * a.N * a.D) : nullptr;
  w.bytes = r.off;
  return w;
}

template <typename T>
void launch_sum_heads(const float* src, T* dst, int B, int heads, int each, int64_t head, hipStream_t st,
                      const Timer& timed) {
  const int64_t total = (int64_t)B * heads * head;
  timed("k_delta_sum_heads", st, [&] {
    hipLaunchKernelGGL(k_delta_sum_heads<T>, dim3((unsigned)((total / 4 + kThr - 1) / kThr)), dim3(kThr), 0, st, src, dst,
                       each, head, total);
  });
}

template <typename T>
void launch_delta_forward(const DeltaArgs& a, const float* state, void* out, float* final_state, void* saved, bool keep,
                          hipStream_t st, const Timer& timed) {
  const int U = a.B * a.Hv, rep = a.H / a.Hv;
  const DeltaSaved s = delta_saved_view(saved, U, a.NC, keep);
  timed("k_delta_chunk", st,
        [&] { hipLaunchKernelGGL(k_delta_chunk<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, s.G, s.T, s.M, s.D); });
  walk<false>(a, s.M, s.D, state, s.S, final_state, s.scratch, false, st, timed);
  // all heads of a state in one block, unless that leaves CUs without one
  const int parts = std::clamp((1024 + U * a.NC - 1) / (U * a.NC), 1, rep), each = (rep + parts - 1) / parts;
  const dim3 grid(U * a.NC * ((rep + each - 1) / each));
  timed("k_delta_out", st, [&] {
    if (keep)
      hipLaunchKernelGGL((k_delta_out<T, true>), grid, dim3(kThr), 0, st, a, each, s.G, s.T, s.S, s.Z,
                         static_cast<T*>(out));
    else
      hipLaunchKernelGGL((k_delta_out<T, false>), grid, dim3(kThr), 0, st, a, each, s.G, s.T, s.S, s.Z,
                         static_cast<T*>(out));
  });
}

template <typename T>
void launch_delta_backward(const DeltaArgs& a, const void* saved, const void* dout, const float* dfinal, void* dq,
                           void* dk, void* dv, float* dg, void* dbeta, float* dstate, void* work, hipStream_t st,
                           const Timer& timed) {
  const int U = a.B * a.Hv;
  const DeltaSaved s = delta_saved_view(const_cast<void*>(saved), U, a.NC, true);
  const DeltaWork w = delta_work_view(work, a);
  const T* od = static_cast<const T*>(dout);
  timed("k_delta_bwd_local", st, [&] {
    hipLaunchKernelGGL(k_delta_bwd_local<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, od, s.G, s.T, w.E, w.F);
  });
  walk<true>(a, s.M, w.F, dfinal, w.dS, dstate, w.scratch, true, st, timed);
  timed("k_delta_bwd_out", st, [&] {
    hipLaunchKernelGGL(k_delta_bwd_out<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, od, s.G, s.T, s.S, s.Z, w.E, w.dS,
                       static_cast<T*>(dq), w.dqh, static_cast<T*>(dk), w.dkh, static_cast<T*>(dv), dg, dbeta);
  });
  if (w.dqh) launch_sum_heads(w.dqh, static_cast<T*>(dq), a.B, a.Hq, a.H / a.Hq, (int64_t)a.N * a.D, st, timed);
  if (w.dkh) launch_sum_heads(w.dkh, static_cast<T*>(dk), a.B, a.Hk, a.Hv / a.Hk, (int64_t)a.N * a.D, st, timed);
}

#define OAL_DELTA(T)                                                                                                 \
  template void launch_sum_heads<T>(const float*, T*, int, int, int, int64_t, hipStream_t, const Timer&);            \
  template void launch_delta_forward<T>(const DeltaArgs&, const float*, void*, float*, void*, bool, hipStream_t,     \
                                        const Timer&);                                                              \
  template void launch_delta_backward<T>(const DeltaArgs&, const void*, const void*, const float*, void*, void*,     \
                                         void*, float*, void*, float*, void*, hipStream_t, const Timer&);
OAL_DELTA(float)
OAL_DELTA(uint16_t)
OAL_DELTA(_Float16)
#undef OAL_DELTA

void launch_delta_step(int kind, const DeltaStepArgs& a, hipStream_t st, const Timer& timed) {
  timed("k_delta_step", st, [&] {
    const dim3 grid(a.B * a.Hv), block(kThr);
    if (kind == 0)
      hipLaunchKernelGGL(k_delta_step<float>, grid, block, 0, st, a);
    else if (kind == 1)
      hipLaunchKernelGGL(k_delta_step<uint16_t>, grid, block, 0, st, a);
    else
      hipLaunchKernelGGL(k_delta_step<_Float16>, grid, block, 0, st, a);
  });
}

}  // namespace oal
