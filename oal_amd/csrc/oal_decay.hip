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
// What makes the state and the decays' gradients is exact to fp32 whatever the tensors'
// type (oal_tile.hpp): a state is a sum over all tokens before it and is handed on in fp32.
//
// Decays enter as differences of sums, held in two floats (48 bits): a token that
// forgets everything (g of -inf, the first of a new text) leaves large sums whose differences still matter.

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
// exp of less is zero in fp32.
constexpr float kNothingKept = -104.f;

// Of a chunk's tokens: log2 of the decay up to and with the token, in two parts; the decay since
// the chunk's start and until its end. end: the chunk's decay, in two parts.
struct alignas(16) Decays {
  float hi[64], lo[64], since[64], until[64], end[4];
};
constexpr int kDecays = sizeof(Decays) / sizeof(float);

__device__ __forceinline__ f32x4 four(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
// Decays from token (hi, lo) to tokens r .. r + 3, and from those to it.
__device__ __forceinline__ f32x4 decay_to(const Decays& s, int r, float hi, float lo) {
  const f32x4 h = four(s.hi + r), l = four(s.lo + r);
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_exp2f((h[i] - hi) + (l[i] - lo));
  return y;
}
__device__ __forceinline__ f32x4 decay_from(const Decays& s, int r, float hi, float lo) {
  const f32x4 h = four(s.hi + r), l = four(s.lo + r);
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_exp2f((hi - h[i]) + (lo - l[i]));
  return y;
}
__device__ __forceinline__ void copy_decays(Decays& s, const Decays& src, int t) {
  if (t < kDecays / 4) reinterpret_cast<float4*>(&s)[t] = reinterpret_cast<const float4*>(&src)[t];
}

__device__ __forceinline__ float gate_at(const DecayArgs& a, int b, int h, int tok) {
  return static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + tok * a.g.n];
}

// The first wave of the block; tokens past N decay nothing.
__device__ __forceinline__ void form_decays(Decays& s, const DecayArgs& a, int b, int h, int tok0, int t) {
  if (t >= 64) return;
  const int tok = tok0 + t;
  double x = 0;
  if (tok < a.N) {
    x = gate_at(a, b, h, tok);
    x = (x < kLeast ? kLeast : x) * 1.4426950408889634;
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
  s.since[t] = __builtin_amdgcn_exp2f(hi + lo);
  s.until[t] = __builtin_amdgcn_exp2f((float)(end - x));
  // slow decays stay for many chunks: their chunks' factors multiply
  const double whole = exp2(end);
  const float first = (float)whole;
  if (t < 4) s.end[t] = t == 0 ? first : t == 1 ? (float)(whole - (double)first) : 0.f;
}

template <typename T>
__device__ __forceinline__ const T* rows_of(const Strided& s, int b, int h, int tok0) {
  return static_cast<const T*>(s.p) + b * s.b + h * s.h + (int64_t)tok0 * s.n;
}

// The column x of a tile of 64 rows, read by rows 32 s + 8 g + j, each row scaled: operand exact to fp32.
template <int NP>
__device__ __forceinline__ Frag<3> scaled_col(const Tile<NP>& s, int c0, int half, int lane, const float* by, float scale) {
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
  return split<3>(v);
}

}  // namespace

// What a chunk adds to the state, D = K^T (e^(G_63 - G) V); its decays. A wave per 16 columns.
template <typename T>
__global__ __launch_bounds__(kThr) void k_decay_sum(DecayArgs a, Decays* __restrict__ G, float* __restrict__ D) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K, V;
  __shared__ Decays dec;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0);
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  Incoming<NP, T> ki, vi;
  ki.fetch(rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
  vi.fetch(rows_of<T>(a.v, b, h, tok0), a.v.n, a.DV, live, t);
  form_decays(dec, a, b, h, tok0, t);
  ki.store(K, t);
  vi.store(V, t);
  lds_sync();
  copy_decays(G[(size_t)u * a.NC + ch], dec, t);
  const Frag<3> v0 = scaled_col(V, 16 * w, 0, lane, dec.until, 1.f), v1 = scaled_col(V, 16 * w, 1, lane, dec.until, 1.f);
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    f32x4 x = mma(col_frag(K, 16 * m, 0, lane), v0, f32x4{});
    x = mma(col_frag(K, 16 * m, 1, lane), v1, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) D[at + (16 * m + 4 * g + i) * 64 + 16 * w + c] = x[i];
  }
}

// S' = e S + D over the chunks, or back over them; what a chunk adds is replaced by the state
// that it starts from (back: whose gradient it takes). Four values per thread.
struct Scan {
  const Decays* G;
  float* S;           // [U][NC][64][64]
  const float* init;  // [U][rows][cols] (null: zero)
  float* end;         // the same (null: not wanted)
  int NC, rows, cols;
  bool back;
};
__global__ __launch_bounds__(kThr) void k_decay_scan(Scan a) {
  const int x = blockIdx.x * kThr + threadIdx.x, u = x >> 10, i = 4 * (x & 1023), row = i >> 6, col = i & 63;
  const bool held = row < a.rows && col < a.cols;
  const size_t slot = ((size_t)u * a.rows + row) * a.cols + col;
  f32x4 s = {};
  if (a.init && held) s = load4(a.init + slot);
  for (int n = 0; n < a.NC; ++n) {
    const size_t at = (size_t)u * a.NC + (a.back ? a.NC - 1 - n : n);
    float* p = a.S + at * kTile2 + i;
    const f32x4 d = load4(p);
    const float hi = a.G[at].end[0], lo = a.G[at].end[1];
    store4(p, s);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = fmaf(hi, s[e], fmaf(lo, s[e], d[e]));
  }
  if (a.end && held) store4(a.end + slot, s);
}

// The outputs of one chunk for `each` output heads of a state head, transposed: a wave's 16 queries
// are the columns, so the scores are an operand of the product with V as they are. 16-bit tensors take
// two parts per value, twice their precision: one rounding is the output's own.
template <typename T>
__global__ __launch_bounds__(kThr) void k_decay_out(DecayArgs a, int each, const Decays* __restrict__ G,
                                                    const float* __restrict__ Sin, T* __restrict__ out) {
  constexpr int NP = kPartsOf<T>, NO = NP == 3 ? 3 : 2;
  __shared__ Tile<NP> K, V;
  __shared__ Tile<NO> S;
  __shared__ Decays dec;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int rep = a.H / a.Hv, parts = (rep + each - 1) / each;
  const int part = blockIdx.x % parts, ch = blockIdx.x / parts % a.NC, u = blockIdx.x / parts / a.NC;
  const int b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  Incoming<NP, T> ki, vi;
  Incoming<NO, float> si;
  ki.fetch(rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, a.D, live, t);
  vi.fetch(rows_of<T>(a.v, b, h, tok0), a.v.n, a.DV, live, t);
  si.fetch(Sin + ((size_t)u * a.NC + ch) * kTile2, 64, 64, 64, t);
  copy_decays(dec, G[(size_t)u * a.NC + ch], t);
  ki.store(K, t);
  vi.store(V, t);
  si.store(S, t);
  lds_sync();
  const float since = a.scale * dec.since[own], hi = dec.hi[own], lo = dec.lo[own];
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
      acc[m] *= since;
      if (m > w) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) p[m] = mma(row_frag(K, 16 * m, s, lane), qf[s], p[m]);
      const f32x4 y = p[m] * a.scale * decay_from(dec, 16 * m + 4 * g, hi, lo);
#pragma unroll
      for (int i = 0; i < 4; ++i) p[m][i] = 16 * m + 4 * g + i <= own ? y[i] : 0.f;
    }
    const Frag<NO> p0 = acc_frag<NO>(p[0], p[1]), p1 = acc_frag<NO>(p[2], p[3]);
    T* dst = out + (((size_t)b * a.H + o) * a.N + tok0 + own) * a.DV;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      acc[m] = mma(col_frag_perm(V, 16 * m, 0, lane), p0, acc[m]);
      if (w >= 2) acc[m] = mma(col_frag_perm(V, 16 * m, 1, lane), p1, acc[m]);
      if (own < live && 16 * m + 4 * g < a.DV) store4(dst + 16 * m + 4 * g, acc[m]);
    }
  }
}

// What a chunk's outputs ask of the state before it, F = scale (e^G Q)^T dO, over a state's output heads.
template <typename T>
__global__ __launch_bounds__(kThr) void k_decay_bwd_sum(DecayArgs a, const T* __restrict__ dout,
                                                        const Decays* __restrict__ G, float* __restrict__ F) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> Q, O;
  __shared__ Decays dec;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0);
  const int each = a.H / a.Hv, o1 = (h + 1) * each;
  Incoming<NP, T> qi, oi;
  auto fetch = [&](int o) {
    qi.fetch(rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0), a.q.n, a.D, live, t);
    oi.fetch(dout + (((size_t)b * a.H + o) * a.N + tok0) * a.DV, a.DV, a.DV, live, t);
  };
  fetch(h * each);
  copy_decays(dec, G[(size_t)u * a.NC + ch], t);
  f32x4 f[4] = {};
  for (int o = h * each; o < o1; ++o) {
    if (o > h * each) lds_sync();
    qi.store(Q, t);
    oi.store(O, t);
    lds_sync();
    if (o + 1 < o1) fetch(o + 1);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const Frag<3> of = scaled_col(O, 16 * w, s, lane, dec.since, a.scale);
#pragma unroll
      for (int m = 0; m < 4; ++m) f[m] = mma(col_frag(Q, 16 * m, s, lane), of, f[m]);
    }
  }
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) F[at + (16 * m + 4 * g + i) * 64 + 16 * w + c] = f[m][i];
}

// All gradients of one chunk and state head, with D_ij = scale exp(G_i - G_j) (j <= i):
//   dq_i = scale e^(G_i) S dO_i + sum_j D_ij (dO_i.v_j) k_j     (per output head)
//   dk_j = e^(G_63 - G_j) dS' v_j + sum_i D_ij (dO_i.v_j) q_i
//   dv_j = e^(G_63 - G_j) dS'^T k_j + sum_i D_ij (q_i.k_j) dO_i
//   dG_i = sum_(j < i) D_ij (q_i.k_j) (dO_i.v_j) - sum_(j > i) D_ji (q_j.k_i) (dO_j.v_i)
//          + scale e^(G_i) q_i.(S dO_i) - e^(G_63 - G_i) k_i.(dS' v_i),
//   and at the chunk's end e^(G_63) <S, dS'> + sum_j e^(G_63 - G_j) k_j.(dS' v_j);
// dg the sums of dG from each token to the chunk's end. Terms that do not decay (j = i,
// the last token's write) are left out rather than cancelled: where all decay is
// strong, dg is far smaller than they are. All products are transposed: a wave's 16
// tokens are the columns. What goes into dq, dk and dv alone is cut to two bf16 parts
// (16 bits) for 16-bit tensors, which then round once themselves; dg sees three.
template <typename T>
__global__ __launch_bounds__(kThr) void k_decay_bwd(DecayArgs a, const T* __restrict__ dout, const Decays* __restrict__ G,
                                                    const float* __restrict__ Sin, const float* __restrict__ dSin,
                                                    T* __restrict__ dq, float* __restrict__ dqh, T* __restrict__ dk,
                                                    float* __restrict__ dkh, T* __restrict__ dv, float* __restrict__ dg,
                                                    double* __restrict__ dgsum) {
  constexpr int NP = kPartsOf<T>, NO = NP == 3 ? 3 : 2;
  __shared__ Tile<NP> K, V, Q, O;
  __shared__ Tile<3> X;
  __shared__ Decays dec;
  __shared__ float dG[64], part[4];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  const T* krows = rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0);
  Incoming<NP, T> ki, vi, qi, oi;
  Incoming<3, float> xi;
  ki.fetch(krows, a.k.n, a.D, live, t);
  vi.fetch(rows_of<T>(a.v, b, h, tok0), a.v.n, a.DV, live, t);
  xi.fetch(dSin + at, 64, 64, 64, t);
  // <S, dS'>
  float ends = 0.f;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = 4 * (t + kThr * x);
    const f32x4 s = load4(Sin + at + i), d = load4(dSin + at + i);
    ends += s[0] * d[0] + s[1] * d[1] + s[2] * d[2] + s[3] * d[3];
  }
  copy_decays(dec, G[(size_t)u * a.NC + ch], t);
  ki.store(K, t);
  vi.store(V, t);
  xi.store(X, t);
  lds_sync();
  xi.fetch(Sin + at, 64, 64, 64, t);
  const int each = a.H / a.Hv, o1 = (h + 1) * each;
  auto fetch = [&](int o) {
    qi.fetch(rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0), a.q.n, a.D, live, t);
    oi.fetch(dout + (((size_t)b * a.H + o) * a.N + tok0) * a.DV, a.DV, a.DV, live, t);
  };
  fetch(h * each);
  ends *= dec.since[63];
  const float hi = dec.hi[own], lo = dec.lo[own];
  Frag<NP> kf[2], vf[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) kf[s] = row_frag(K, 16 * w, s, lane), vf[s] = row_frag(V, 16 * w, s, lane);
  f32x4 wk[4], wv[4];  // dk and dv
  float decay = 0.f;   // of dG
  {
    const float until = dec.until[own];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      f32x4 kv = {}, x = {}, y = {};
      if (own < live && 16 * n + 4 * g < a.D) kv = load4(krows + own * a.k.n + 16 * n + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        x = mma(row_frag(X, 16 * n, s, lane), vf[s], x);
        y = mma(col_frag<NO>(X, 16 * n, s, lane), kf[s], y);
      }
      wk[n] = until * x;
      wv[n] = until * y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // what the last token writes does not decay
        const float z = own < live - 1 ? kv[i] * wk[n][i] : 0.f;
        ends += z;
        decay -= z;
      }
    }
  }
  ends = wave_sum(ends);
  if (lane == 0) part[w] = ends;
  lds_sync();
  xi.store(X, t);
  const float since = a.scale * dec.since[own];
  for (int o = h * each; o < o1; ++o) {
    const T* qrows = rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0);
    const size_t orow = ((size_t)b * a.H + o) * a.N + tok0;
    if (o > h * each) lds_sync();
    qi.store(Q, t);
    oi.store(O, t);
    lds_sync();
    if (o + 1 < o1) fetch(o + 1);
    Frag<NP> of[2], qf[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) of[s] = row_frag(O, 16 * w, s, lane), qf[s] = row_frag(Q, 16 * w, s, lane);
    f32x4 acc[4], p[4] = {};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      f32x4 x = {}, qk = {}, qv = {};
      if (own < live && 16 * n + 4 * g < a.D) qv = load4(qrows + own * a.q.n + 16 * n + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s) x = mma(row_frag(X, 16 * n, s, lane), of[s], x);
      acc[n] = since * x;
#pragma unroll
      for (int i = 0; i < 4; ++i) decay += qv[i] * acc[n][i];
      if (n > w) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        p[n] = mma(row_frag(V, 16 * n, s, lane), of[s], p[n]);
        qk = mma(row_frag(K, 16 * n, s, lane), qf[s], qk);
      }
      const f32x4 y = a.scale * decay_from(dec, 16 * n + 4 * g, hi, lo) * p[n];
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
    f32x4 r[4] = {};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      p[n] = f32x4{};
      if (n < w) continue;
      f32x4 qk = {}, ov = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        ov = mma(row_frag(O, 16 * n, s, lane), vf[s], ov);
        qk = mma(row_frag(Q, 16 * n, s, lane), kf[s], qk);
      }
      const f32x4 y = a.scale * decay_to(dec, 16 * n + 4 * g, hi, lo);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * n + 4 * g + i;
        const float e = own <= row ? y[i] : 0.f;
        p[n][i] = e * ov[i];
        r[n][i] = e * qk[i];
        decay -= own < row ? p[n][i] * qk[i] : 0.f;
      }
    }
    const Frag<NO> p0 = acc_frag<NO>(p[0], p[1]), p1 = acc_frag<NO>(p[2], p[3]);
    const Frag<NO> r0 = acc_frag<NO>(r[0], r[1]), r1 = acc_frag<NO>(r[2], r[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (w < 2) {
        wk[n] = mma(col_frag_perm(Q, 16 * n, 0, lane), p0, wk[n]);
        wv[n] = mma(col_frag_perm(O, 16 * n, 0, lane), r0, wv[n]);
      }
      wk[n] = mma(col_frag_perm(Q, 16 * n, 1, lane), p1, wk[n]);
      wv[n] = mma(col_frag_perm(O, 16 * n, 1, lane), r1, wv[n]);
    }
  }
  const size_t row = (size_t)u * a.N + tok0 + own;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int d = 16 * n + 4 * g;
    if (own < live && d < a.D) {
      if (dkh)
        store4(dkh + row * a.D + d, wk[n]);
      else
        store4(dk + row * a.D + d, wk[n]);
    }
    if (own < live && d < a.DV) store4(dv + row * a.DV + d, wv[n]);
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
    // where nothing is kept nothing depends on g; the sums' roundings do not cancel
    if (lane >= live || gate_at(a, b, h, tok0 + lane) < kNothingKept) x = 0;
    if (dgsum) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
      if (lane == 0) dgsum[(size_t)u * a.NC + ch] = x;
    } else if (lane < live) {
      dg[(size_t)u * a.N + tok0 + lane] = (float)x;
    }
  }
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

void scan(const DecayArgs& a, const float* G, float* S, const float* init, float* end, bool back, hipStream_t st,
          const Timer& timed) {
  const Scan s = {reinterpret_cast<const Decays*>(G), S, init, end, a.NC, a.D, a.DV, back};
  timed("k_decay_scan", st, [&] { hipLaunchKernelGGL(k_decay_scan, dim3(4 * a.B * a.Hv), dim3(kThr), 0, st, s); });
}
}  // namespace

DecaySaved decay_saved_view(void* base, int U, int NC) {
  DecaySaved s;
  Room r{static_cast<char*>(base)};
  s.G = r.take<float>((size_t)U * NC * kDecays);
  s.S = r.take<float>((size_t)U * NC * kTile2);
  s.bytes = r.off;
  return s;
}

DecayWork decay_work_view(void* base, const DecayArgs& a) {
  DecayWork w;
  Room r{static_cast<char*>(base)};
  const size_t chunks = (size_t)a.B * a.Hv * a.NC;
  w.dS = r.take<float>(chunks * kTile2);
  w.dqh = a.H != a.Hq ? r.take<float>((size_t)a.B * a.H * a.N * a.D) : nullptr;
  w.dkh = a.Hv != a.Hk ? r.take<float>((size_t)a.B * a.Hv * a.N * a.D) : nullptr;
  w.sum = a.per_head ? r.take<double>(chunks) : nullptr;
  w.bytes = r.off;
  return w;
}

template <typename T>
void launch_decay_forward(const DecayArgs& a, const float* state, void* out, float* final_state, void* saved,
                          hipStream_t st, const Timer& timed) {
  const int U = a.B * a.Hv, rep = a.H / a.Hv;
  const DecaySaved s = decay_saved_view(saved, U, a.NC);
  Decays* G = reinterpret_cast<Decays*>(s.G);
  timed("k_decay_sum", st,
        [&] { hipLaunchKernelGGL(k_decay_sum<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, G, s.S); });
  scan(a, s.G, s.S, state, final_state, false, st, timed);
  // all heads of a state in one block, unless that leaves CUs without one
  const int parts = std::clamp((1024 + U * a.NC - 1) / (U * a.NC), 1, rep), each = (rep + parts - 1) / parts;
  timed("k_decay_out", st, [&] {
    hipLaunchKernelGGL(k_decay_out<T>, dim3(U * a.NC * ((rep + each - 1) / each)), dim3(kThr), 0, st, a, each, G, s.S,
                       static_cast<T*>(out));
  });
}

template <typename T>
void launch_decay_backward(const DecayArgs& a, const void* saved, const void* dout, const float* dfinal, void* dq,
                           void* dk, void* dv, float* dg, float* dstate, void* work, hipStream_t st,
                           const Timer& timed) {
  const int U = a.B * a.Hv;
  const DecaySaved s = decay_saved_view(const_cast<void*>(saved), U, a.NC);
  const DecayWork w = decay_work_view(work, a);
  const Decays* G = reinterpret_cast<const Decays*>(s.G);
  const T* od = static_cast<const T*>(dout);
  timed("k_decay_bwd_sum", st,
        [&] { hipLaunchKernelGGL(k_decay_bwd_sum<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, od, G, w.dS); });
  scan(a, s.G, w.dS, dfinal, dstate, true, st, timed);
  timed("k_decay_bwd", st, [&] {
    hipLaunchKernelGGL(k_decay_bwd<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, od, G, s.S, w.dS, static_cast<T*>(dq),
                       w.dqh, static_cast<T*>(dk), w.dkh, static_cast<T*>(dv), dg, w.sum);
  });
  if (w.sum)
    timed("k_decay_gate_sum", st, [&] {
      hipLaunchKernelGGL(k_decay_gate_sum, dim3(a.Hv), dim3(kThr), 0, st, w.sum, a.B, a.Hv, a.NC, dg);
    });
  if (w.dqh) launch_sum_heads(w.dqh, static_cast<T*>(dq), a.B, a.Hq, a.H / a.Hq, (int64_t)a.N * a.D, st, timed);
  if (w.dkh) launch_sum_heads(w.dkh, static_cast<T*>(dk), a.B, a.Hk, a.Hv / a.Hk, (int64_t)a.N * a.D, st, timed);
}

#define OAL_DECAY(T)                                                                                               \
  template void launch_decay_forward<T>(const DecayArgs&, const float*, void*, float*, void*, hipStream_t,         \
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
