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
// T and O are formed chunk by chunk at once, S and Z in a walk over the chunks.
// The walk's products are exact to fp32 whatever the tensors' type (oal_tile.hpp):
// a state is a sum over all tokens before it and is handed on in fp32.
//
// Decays enter as differences of sums, held in two floats (48 bits): a token that
// forgets nearly everything leaves large sums whose differences still matter.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oal_common.hpp"
#include "oal_delta.hpp"
#include "oal_tile.hpp"

namespace oal {

namespace {

constexpr int kThr = 256;
constexpr int kTile2 = 64 * 64;
// Smallest log-decay: exp of it is zero, and 64 of them leave the sums' differences exact.
constexpr double kLeast = -1e4;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct Gates {
  float hi[64], lo[64], beta[64];  // log2 of the decay up to and with token i, in two parts
  __device__ float between(int i, int j) const {
    return __builtin_amdgcn_exp2f((hi[i] - hi[j]) + (lo[i] - lo[j]));
  }
  __device__ float since(int i) const { return __builtin_amdgcn_exp2f(hi[i] + lo[i]); }
};

__device__ __forceinline__ float beta_at(const DeltaArgs& a, int b, int h, int tok, bool bf16) {
  const int64_t at = b * a.beta.b + h * a.beta.h + tok * a.beta.n;
  return bf16 && !a.beta32 ? to_f(static_cast<const uint16_t*>(a.beta.p)[at]) : static_cast<const float*>(a.beta.p)[at];
}

// The first wave of the block; tokens past N decay nothing and write nothing.
template <typename T>
__device__ __forceinline__ void load_gates(Gates& s, const DeltaArgs& a, int b, int h, int tok0, int t) {
  if (t >= 64) return;
  const int tok = tok0 + t;
  double x = 0;
  float beta = 0;
  if (tok < a.N) {
    x = static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + tok * a.g.n];
    x = (x < kLeast ? kLeast : x) * 1.4426950408889634;
    beta = beta_at(a, b, h, tok, sizeof(T) == 2);
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __shfl_up(x, off, 64);
    if (t >= off) x += y;
  }
  s.hi[t] = (float)x;
  s.lo[t] = (float)(x - (double)(float)x);
  s.beta[t] = beta;
}

template <typename T>
__device__ __forceinline__ const T* rows_of(const Strided& s, int b, int h, int tok0) {
  return static_cast<const T*>(s.p) + b * s.b + h * s.h + (int64_t)tok0 * s.n;
}

// 64 x 64 fp32 values into NP parts.
template <int NP>
__device__ __forceinline__ void load_f32(Tile<NP>& s, const float* __restrict__ src, int t) {
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = t + kThr * x;
    float v[8];
    load_row8(v, src + 8 * i);
    const Frag<NP> f = split<NP>(v);
#pragma unroll
    for (int e = 0; e < NP; ++e)
      *reinterpret_cast<bf16x8*>(s.x + e * kTileElems + (i >> 3) * kTileRow + 8 * (i & 7)) = f.p[e];
  }
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

// T of one chunk. Diagonal blocks of 16 rows by substitution (a lane per
// column), then twice the rule for two blocks, [L11 0; L21 L22]^-1 =
// [T11 0; -T22 L21 T11, T22], on the fp32 matrix cores.
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_solve(DeltaArgs a, uint16_t* __restrict__ out) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K;
  __shared__ Gates gate;
  __shared__ alignas(16) float L[64 * kRow32], S[64 * kRow32], Y[32 * kRow32];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0);
  load_gates<T>(gate, a, b, h, tok0, t);
  load_tile<64, kThr>(K, rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, live, t);
  __syncthreads();
  for (int n = 0; n < 4; ++n) {
    f32x4 kk = {};
    if (n <= w)
      for (int s = 0; s < 2; ++s) kk = mma(row_frag(K, 16 * w, s, lane), row_frag(K, 16 * n, s, lane), kk);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * w + 4 * g + r, j = 16 * n + c;
      L[i * kRow32 + j] = j < i ? kk[r] * gate.between(i, j) * gate.beta[j] : 0.f;
      S[i * kRow32 + j] = 0.f;
    }
  }
  __syncthreads();
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
  __syncthreads();
  f32x4 y = {};
  if (w < 2) {
    const int o = 32 * w;
    y = mma_f32<16>(L + (o + 16) * kRow32 + o, S + o * kRow32 + o, y, lane);
#pragma unroll
    for (int r = 0; r < 4; ++r) Y[(16 * w + 4 * g + r) * kRow32 + c] = y[r];
  }
  __syncthreads();
  if (w < 2) {
    const int o = 32 * w;
    y = mma_f32<16>(S + (o + 16) * kRow32 + o + 16, Y + 16 * w * kRow32, f32x4{}, lane);
#pragma unroll
    for (int r = 0; r < 4; ++r) S[(o + 16 + 4 * g + r) * kRow32 + o + c] = -y[r];
  }
  __syncthreads();
  const int m = 16 * (w >> 1), n = 16 * (w & 1);
  y = mma_f32<32>(L + (32 + m) * kRow32, S + n, f32x4{}, lane);
#pragma unroll
  for (int r = 0; r < 4; ++r) Y[(m + 4 * g + r) * kRow32 + n + c] = y[r];
  __syncthreads();
  y = mma_f32<32>(S + (32 + m) * kRow32 + 32, Y + n, f32x4{}, lane);
#pragma unroll
  for (int r = 0; r < 4; ++r) S[(32 + m + 4 * g + r) * kRow32 + n + c] = -y[r];
  __syncthreads();
  uint16_t* dst = out + ((size_t)u * a.NC + ch) * 3 * kTile2;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int i = t + kThr * x;
    float v[8];
    load_row8(v, S + (i >> 3) * kRow32 + 8 * (i & 7));
    const Frag<3> f = split<3>(v);
#pragma unroll
    for (int e = 0; e < 3; ++e) *reinterpret_cast<bf16x8*>(dst + e * kTile2 + 8 * i) = f.p[e];
  }
}

// The walk over the chunks: a block per unit, a wave per 16 columns of the state,
// whose products stay in its registers.
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_scan(DeltaArgs a, const uint16_t* __restrict__ Tm,
                                                     const float* __restrict__ state, float* __restrict__ Sout,
                                                     float* __restrict__ Zout, float* __restrict__ final_state) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K;
  __shared__ Tile<3> M;
  __shared__ Gates gate;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, col = 16 * w + (lane & 15);
  const int u = blockIdx.x, b = u / a.Hv, h = u % a.Hv;
  f32x4 S[4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) S[m][i] = state ? state[(size_t)u * kTile2 + (16 * m + 4 * g + i) * 64 + col] : 0.f;
  for (int ch = 0; ch < a.NC; ++ch) {
    const int tok0 = 64 * ch, live = min(64, a.N - tok0);
    const size_t at = ((size_t)u * a.NC + ch) * kTile2;
    __syncthreads();
    load_gates<T>(gate, a, b, h, tok0, t);
    load_tile<64, kThr>(K, rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, live, t);
#pragma unroll
    for (int x = 0; x < 6; ++x) {
      const int i = t + kThr * x;
      *reinterpret_cast<uint4*>(M.x + (i >> 9) * kTileElems + ((i & 511) >> 3) * kTileRow + 8 * (i & 7)) =
          reinterpret_cast<const uint4*>(Tm + 3 * at)[i];
    }
    const T* v = rows_of<T>(a.v, b, h, tok0);
    f32x4 r[4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * m + 4 * g + i;
        r[m][i] = row < live ? to_f(v[row * a.v.n + col]) : 0.f;
        Sout[at + row * 64 + col] = S[m][i];
      }
    __syncthreads();
    {
      const Frag<3> s0 = acc_frag<3>(S[0], S[1]), s1 = acc_frag<3>(S[2], S[3]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        f32x4 x = mma(row_frag_perm(K, 16 * m, 0, lane), s0, f32x4{});
        x = mma(row_frag_perm(K, 16 * m, 1, lane), s1, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[m][i] -= gate.since(16 * m + 4 * g + i) * x[i];
      }
    }
    f32x4 z[4];
    {
      const Frag<3> r0 = acc_frag<3>(r[0], r[1]), r1 = acc_frag<3>(r[2], r[3]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        z[m] = mma(row_frag_perm(M, 16 * m, 0, lane), r0, f32x4{});
        if (m >= 2) z[m] = mma(row_frag_perm(M, 16 * m, 1, lane), r1, z[m]);
      }
    }
    const float last = gate.since(63);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * m + 4 * g + i;
        Zout[at + row * 64 + col] = z[m][i];
        z[m][i] *= gate.beta[row] * gate.between(63, row);
        S[m][i] *= last;
      }
    const Frag<3> u0 = acc_frag<3>(z[0], z[1]), u1 = acc_frag<3>(z[2], z[3]);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      S[m] = mma(col_frag_perm(K, 16 * m, 0, lane), u0, S[m]);
      S[m] = mma(col_frag_perm(K, 16 * m, 1, lane), u1, S[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) final_state[(size_t)u * kTile2 + (16 * m + 4 * g + i) * 64 + col] = S[m][i];
}

// Four consecutive values of a row.
__device__ __forceinline__ void store4(float* p, const f32x4& x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void store4(uint16_t* p, const f32x4& x) {
  uint2 v = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  *reinterpret_cast<uint2*>(p) = v;
}
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4 load4(const uint16_t* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
               __uint_as_float(v.y & 0xffff0000u)};
}

// The outputs of one chunk and output head, transposed: a wave's 16 queries are
// the columns, so the scores are an operand of the product with U as they are. The
// scores, U and S enter in the output's own precision.
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_out(DeltaArgs a, const float* __restrict__ Sin,
                                                    const float* __restrict__ Zin, T* __restrict__ out) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K, U, S;
  __shared__ Gates gate;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, b = blockIdx.x / a.NC / a.H, o = blockIdx.x / a.NC % a.H;
  const int h = o / (a.H / a.Hv), u = b * a.Hv + h;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), qrow = 16 * w + c;
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  load_gates<T>(gate, a, b, h, tok0, t);
  load_tile<64, kThr>(K, rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, live, t);
  load_f32(U, Zin + at, t);
  load_f32(S, Sin + at, t);
  const T* q = rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0) + qrow * a.q.n;
  Frag<NP> qf[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) qf[s] = global_frag<NP>(q + 32 * s + 8 * g, qrow < live);
  __syncthreads();
  f32x4 acc[4] = {}, p[4] = {};
  const float since = a.scale * gate.since(qrow);
#pragma unroll
  for (int m = 0; m < 4; ++m) {
#pragma unroll
    for (int s = 0; s < 2; ++s) acc[m] = mma(col_frag(S, 16 * m, s, lane), qf[s], acc[m]);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[m][i] *= since;
    if (m > w) continue;
#pragma unroll
    for (int s = 0; s < 2; ++s) p[m] = mma(row_frag(K, 16 * m, s, lane), qf[s], p[m]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = 16 * m + 4 * g + i;
      p[m][i] = j <= qrow ? p[m][i] * a.scale * gate.between(qrow, j) * gate.beta[j] : 0.f;
    }
  }
  const Frag<NP> p0 = acc_frag<NP>(p[0], p[1]), p1 = acc_frag<NP>(p[2], p[3]);
  T* dst = out + (((size_t)b * a.H + o) * a.N + tok0 + qrow) * 64;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    acc[m] = mma(col_frag_perm(U, 16 * m, 0, lane), p0, acc[m]);
    if (w >= 2) acc[m] = mma(col_frag_perm(U, 16 * m, 1, lane), p1, acc[m]);
    if (qrow < live) store4(dst + 16 * m + 4 * g, acc[m]);
  }
}

// ---------------------------------------------------------------------------
// Backward. Gradients of a chunk's u and of the state before it from its own outputs
// (E, F), at once; then the walk back:
//   dU = E + e^(G_63 - G) K dS',  dZ = T^T (beta dU),
//   dS = F + e^(G_63) dS' - K^T (e^G dZ)
// and from dZ = dV, dU, dS', S and Z everything else of the chunk at once.
// Decays' gradients are sums of terms that cancel, so all of it is exact to fp32.
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_bwd_local(DeltaArgs a, const T* __restrict__ dout,
                                                          float* __restrict__ E, float* __restrict__ F) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> Q, O;
  __shared__ Gates gate;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  load_gates<T>(gate, a, b, h, tok0, t);
  const T* k = rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0) + own * a.k.n;
  Frag<NP> kf[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) kf[s] = global_frag<NP>(k + 32 * s + 8 * g, own < live);
  f32x4 e[4] = {}, f[4] = {};
  const int each = a.H / a.Hv;
  for (int o = h * each; o < (h + 1) * each; ++o) {
    __syncthreads();
    load_tile<64, kThr>(Q, rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0), a.q.n, live, t);
    load_tile<64, kThr>(O, dout + (((size_t)b * a.H + o) * a.N + tok0) * 64, (int64_t)64, live, t);
    __syncthreads();
    f32x4 p[4] = {};
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (m < w) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) p[m] = mma(row_frag(Q, 16 * m, s, lane), kf[s], p[m]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * m + 4 * g + i;
        p[m][i] = own <= row ? p[m][i] * a.scale * gate.between(row, own) : 0.f;
      }
    }
    const Frag<3> p0 = acc_frag<3>(p[0], p[1]), p1 = acc_frag<3>(p[2], p[3]);
    Frag<3> of[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const Frag<NP> x = col_frag(O, 16 * w, s, lane);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = static_cast<float>(x.p[0][j]);
        if constexpr (NP == 3) v[j] = (v[j] + static_cast<float>(x.p[1][j])) + static_cast<float>(x.p[2][j]);
        v[j] *= a.scale * gate.since(32 * s + 8 * g + j);
      }
      of[s] = split<3>(v);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (w < 2) e[m] = mma(col_frag_perm(O, 16 * m, 0, lane), p0, e[m]);
      e[m] = mma(col_frag_perm(O, 16 * m, 1, lane), p1, e[m]);
#pragma unroll
      for (int s = 0; s < 2; ++s) f[m] = mma(col_frag(Q, 16 * m, s, lane), of[s], f[m]);
    }
  }
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    store4(E + at + own * 64 + 16 * m + 4 * g, e[m]);
#pragma unroll
    for (int i = 0; i < 4; ++i) F[at + (16 * m + 4 * g + i) * 64 + 16 * w + c] = f[m][i];
  }
}

template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_bwd_scan(DeltaArgs a, const uint16_t* __restrict__ Tm,
                                                         const float* __restrict__ dfinal, float* __restrict__ E,
                                                         const float* __restrict__ F, float* __restrict__ dSout,
                                                         float* __restrict__ dZout, float* __restrict__ dstate) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K;
  __shared__ Tile<3> M;
  __shared__ Gates gate;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, col = 16 * w + (lane & 15);
  const int u = blockIdx.x, b = u / a.Hv, h = u % a.Hv;
  f32x4 S[4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) S[m][i] = dfinal ? dfinal[(size_t)u * kTile2 + (16 * m + 4 * g + i) * 64 + col] : 0.f;
  for (int ch = a.NC - 1; ch >= 0; --ch) {
    const int tok0 = 64 * ch, live = min(64, a.N - tok0);
    const size_t at = ((size_t)u * a.NC + ch) * kTile2;
    __syncthreads();
    load_gates<T>(gate, a, b, h, tok0, t);
    load_tile<64, kThr>(K, rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0), a.k.n, live, t);
#pragma unroll
    for (int x = 0; x < 6; ++x) {
      const int i = t + kThr * x;
      *reinterpret_cast<uint4*>(M.x + (i >> 9) * kTileElems + ((i & 511) >> 3) * kTileRow + 8 * (i & 7)) =
          reinterpret_cast<const uint4*>(Tm + 3 * at)[i];
    }
    f32x4 r[4], f[4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t x = at + (16 * m + 4 * g + i) * 64 + col;
        r[m][i] = E[x];
        f[m][i] = F[x];
        dSout[x] = S[m][i];
      }
    __syncthreads();
    {
      const Frag<3> s0 = acc_frag<3>(S[0], S[1]), s1 = acc_frag<3>(S[2], S[3]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        f32x4 x = mma(row_frag_perm(K, 16 * m, 0, lane), s0, f32x4{});
        x = mma(row_frag_perm(K, 16 * m, 1, lane), s1, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 16 * m + 4 * g + i;
          r[m][i] += gate.between(63, row) * x[i];
          E[at + row * 64 + col] = r[m][i];
          r[m][i] *= gate.beta[row];
        }
      }
    }
    f32x4 z[4];
    {
      const Frag<3> r0 = acc_frag<3>(r[0], r[1]), r1 = acc_frag<3>(r[2], r[3]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        z[m] = mma(col_frag_perm(M, 16 * m, 1, lane), r1, f32x4{});
        if (m < 2) z[m] = mma(col_frag_perm(M, 16 * m, 0, lane), r0, z[m]);
      }
    }
    const float last = gate.since(63);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * m + 4 * g + i;
        dZout[at + row * 64 + col] = z[m][i];
        z[m][i] *= -gate.since(row);
        S[m][i] = S[m][i] * last + f[m][i];
      }
    const Frag<3> u0 = acc_frag<3>(z[0], z[1]), u1 = acc_frag<3>(z[2], z[3]);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      S[m] = mma(col_frag_perm(K, 16 * m, 0, lane), u0, S[m]);
      S[m] = mma(col_frag_perm(K, 16 * m, 1, lane), u1, S[m]);
    }
  }
  if (dstate) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) dstate[(size_t)u * kTile2 + (16 * m + 4 * g + i) * 64 + col] = S[m][i];
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
// tokens are the columns.
template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_bwd_out(DeltaArgs a, const T* __restrict__ dout,
                                                        const float* __restrict__ Sin, const float* __restrict__ Zin,
                                                        const float* __restrict__ dU, const float* __restrict__ dSin,
                                                        const float* __restrict__ dZ, T* __restrict__ dq,
                                                        float* __restrict__ dqh, T* __restrict__ dk,
                                                        float* __restrict__ dkh, T* __restrict__ dv,
                                                        float* __restrict__ dg, void* __restrict__ dbeta) {
  constexpr int NP = kPartsOf<T>;
  __shared__ Tile<NP> K, Q, O;
  __shared__ Tile<3> Z, X;
  __shared__ Gates gate;
  __shared__ float dG[64], part[4];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int ch = blockIdx.x % a.NC, u = blockIdx.x / a.NC, b = u / a.Hv, h = u % a.Hv;
  const int tok0 = 64 * ch, live = min(64, a.N - tok0), own = 16 * w + c;
  const size_t at = ((size_t)u * a.NC + ch) * kTile2;
  load_gates<T>(gate, a, b, h, tok0, t);
  const T* krows = rows_of<T>(a.k, b, h / (a.Hv / a.Hk), tok0);
  load_tile<64, kThr>(K, krows, a.k.n, live, t);
  load_f32(Z, Zin + at, t);
  load_f32(X, dZ + at, t);
  Frag<3> zf[2], dzf[2];
  own_row(zf, Zin + at + own * 64, g);
  own_row(dzf, dZ + at + own * 64, g);
  __syncthreads();
  const float beta = gate.beta[own];
  f32x4 reads[4] = {}, writes[4] = {};
  float dot = 0.f;    // of dbeta
  float decay = 0.f;  // of dG
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
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 16 * n + 4 * g + i;
        m[n][i] = j < own ? -gate.beta[j] * gate.between(own, j) * m[n][i] : 0.f;
        decay += m[n][i] * kk[i];
      }
    }
    const Frag<3> m0 = acc_frag<3>(m[0], m[1]), m1 = acc_frag<3>(m[2], m[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      reads[n] = mma(col_frag_perm(K, 16 * n, 0, lane), m0, reads[n]);
      if (w >= 2) reads[n] = mma(col_frag_perm(K, 16 * n, 1, lane), m1, reads[n]);
    }
  }
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
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * n + 4 * g + i;
        const float x = own < row ? gate.between(row, own) * m[n][i] : 0.f;
        dot -= x * kk[i];
        m[n][i] = -beta * x;
        decay -= m[n][i] * kk[i];
      }
    }
    const Frag<3> m0 = acc_frag<3>(m[0], m[1]), m1 = acc_frag<3>(m[2], m[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (w < 2) writes[n] = mma(col_frag_perm(K, 16 * n, 0, lane), m0, writes[n]);
      writes[n] = mma(col_frag_perm(K, 16 * n, 1, lane), m1, writes[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int x = own * 64 + 16 * n + 4 * g;
    const f32x4 du = load4(dU + at + x), z = load4(Zin + at + x), dz = load4(dZ + at + x);
#pragma unroll
    for (int i = 0; i < 4; ++i) dot += du[i] * z[i];
    if (own < live) store4(dv + ((size_t)u * a.N + tok0) * 64 + x, dz);
  }
  dot = group_sum(dot);
  if (g == 0 && own < live) {
    const size_t x = (size_t)u * a.N + tok0 + own;
    if (sizeof(T) == 2 && !a.beta32)
      static_cast<uint16_t*>(dbeta)[x] = from_f<uint16_t>(dot);
    else
      static_cast<float*>(dbeta)[x] = dot;
  }
  // the state after the chunk: its share of dk, and <S', dS'>
  __syncthreads();
  load_f32(X, dSin + at, t);
  float ends = 0.f;
  {
    const float last = gate.since(63);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = 4 * (t + kThr * x);
      const f32x4 s = load4(Sin + at + i), d = load4(dSin + at + i);
      ends += last * (s[0] * d[0] + s[1] * d[1] + s[2] * d[2] + s[3] * d[3]);
    }
  }
  __syncthreads();
  f32x4 kv[4];
  {
    const float until = beta * gate.between(63, own);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      kv[n] = f32x4{};
      if (own < live) kv[n] = load4(krows + own * a.k.n + 16 * n + 4 * g);
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
  __syncthreads();
  load_f32(X, Sin + at, t);
  __syncthreads();
  const float since = gate.since(own);
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
  const int each = a.H / a.Hv;
  for (int o = h * each; o < (h + 1) * each; ++o) {
    if (o > h * each) __syncthreads();
    const T* qrows = rows_of<T>(a.q, b, o / (a.H / a.Hq), tok0);
    const size_t orow = ((size_t)b * a.H + o) * a.N + tok0;
    load_tile<64, kThr>(Q, qrows, a.q.n, live, t);
    load_tile<64, kThr>(O, dout + orow * 64, (int64_t)64, live, t);
    __syncthreads();
    Frag<NP> of[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) of[s] = row_frag(O, 16 * w, s, lane);
    f32x4 acc[4], p[4] = {};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      f32x4 x = {}, qk = {}, qv = {};
      if (own < live) qv = load4(qrows + own * a.q.n + 16 * n + 4 * g);
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
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 16 * n + 4 * g + i;
        p[n][i] = j <= own ? a.scale * gate.beta[j] * gate.between(own, j) * p[n][i] : 0.f;
        if (j < own) decay += p[n][i] * qk[i];
      }
    }
    {
      const Frag<3> p0 = acc_frag<3>(p[0], p[1]), p1 = acc_frag<3>(p[2], p[3]);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        acc[n] = mma(col_frag_perm(K, 16 * n, 0, lane), p0, acc[n]);
        if (w >= 2) acc[n] = mma(col_frag_perm(K, 16 * n, 1, lane), p1, acc[n]);
        if (own < live) {
          if (dqh)
            store4(dqh + (orow + own) * 64 + 16 * n + 4 * g, acc[n]);
          else
            store4(dq + (orow + own) * 64 + 16 * n + 4 * g, acc[n]);
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
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * n + 4 * g + i;
        p[n][i] = own <= row ? a.scale * beta * gate.between(row, own) * p[n][i] : 0.f;
        if (own < row) decay -= p[n][i] * qk[i];
      }
    }
    const Frag<3> p0 = acc_frag<3>(p[0], p[1]), p1 = acc_frag<3>(p[2], p[3]);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (w < 2) writes[n] = mma(col_frag_perm(Q, 16 * n, 0, lane), p0, writes[n]);
      writes[n] = mma(col_frag_perm(Q, 16 * n, 1, lane), p1, writes[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (own < live) {
      const f32x4 x = reads[n] + writes[n];
      const size_t row = ((size_t)u * a.N + tok0 + own) * 64 + 16 * n + 4 * g;
      if (dkh)
        store4(dkh + row, x);
      else
        store4(dk + row, x);
    }
  }
  decay = group_sum(decay);
  if (g == 0) dG[own] = decay;
  __syncthreads();
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
// [B][heads][N][64] of src [B][heads each][N][64].
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
// state, 4 x 4 values per thread, for all N tokens and writes it back.
// ---------------------------------------------------------------------------
namespace {
__device__ __forceinline__ float value(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float value(const uint16_t* p, int64_t i) { return to_f(p[i]); }
__device__ __forceinline__ float value(const _Float16* p, int64_t i) { return static_cast<float>(p[i]); }
__device__ __forceinline__ void put(float* p, int64_t i, float x) { p[i] = x; }
__device__ __forceinline__ void put(uint16_t* p, int64_t i, float x) { p[i] = from_f<uint16_t>(x); }
__device__ __forceinline__ void put(_Float16* p, int64_t i, float x) { p[i] = static_cast<_Float16>(x); }
}  // namespace

template <typename T>
__global__ __launch_bounds__(kThr) void k_delta_step(DeltaStepArgs a) {
  __shared__ float sum[4][64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int u = blockIdx.x, b = u / a.Hv, h = u % a.Hv;
  const int d0 = 4 * (t >> 4), c0 = 4 * (t & 15);
  float* state = a.state + (size_t)u * a.Dk * a.Dv;
  float s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      s[i][j] = d0 + i < a.Dk && c0 + j < a.Dv ? state[(d0 + i) * a.Dv + c0 + j] : 0.f;
  const T* k = static_cast<const T*>(a.k.p) + b * a.k.b + (h / (a.Hv / a.Hk)) * a.k.h;
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.b + h * a.v.h;
  const int each = a.H / a.Hv;
  // sums over the rows of x[4] per column, all columns c0 .. c0 + 3 of this thread
  auto over_rows = [&](float (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = group_sum(x[j]);
    __syncthreads();
    if (lane < 16)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[w][c0 + j] = x[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (sum[0][c0 + j] + sum[1][c0 + j]) + (sum[2][c0 + j] + sum[3][c0 + j]);
  };
  for (int n = 0; n < a.N; ++n) {
    const float decay = expf(static_cast<const float*>(a.g.p)[b * a.g.b + h * a.g.h + n * a.g.n]);
    const int64_t bx = b * a.beta.b + h * a.beta.h + n * a.beta.n;
    const float beta = a.beta32 ? static_cast<const float*>(a.beta.p)[bx] : value(static_cast<const T*>(a.beta.p), bx);
    float kr[4], x[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kr[i] = d0 + i < a.Dk ? value(k, n * a.k.n + d0 + i) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] *= decay;
        x[j] += kr[i] * s[i][j];
      }
    }
    over_rows(x);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float vj = c0 + j < a.Dv ? value(v, n * a.v.n + c0 + j) : 0.f;
      const float uj = beta * (vj - x[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i][j] += kr[i] * uj;
    }
    for (int o = h * each; o < (h + 1) * each; ++o) {
      const T* q = static_cast<const T*>(a.q.p) + b * a.q.b + (o / (a.H / a.Hq)) * a.q.h + n * a.q.n;
      float y[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float qi = d0 + i < a.Dk ? value(q, d0 + i) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += qi * s[i][j];
      }
      over_rows(y);
      T* out = static_cast<T*>(a.out) + (((size_t)b * a.H + o) * a.N + n) * a.Dv;
      if (t < 16)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c0 + j < a.Dv) put(out, c0 + j, a.scale * y[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d0 + i < a.Dk && c0 + j < a.Dv) state[(d0 + i) * a.Dv + c0 + j] = s[i][j];
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
DeltaSaved delta_saved_view(void* base, int U, int NC) {
  DeltaSaved s;
  size_t off = 0;
  const size_t tiles = (size_t)U * NC * kTile2;
  auto take = [&](size_t bytes) {
    char* p = static_cast<char*>(base) + off;
    off += align256(bytes);
    return p;
  };
  s.T = reinterpret_cast<uint16_t*>(take(tiles * 6));
  s.S = reinterpret_cast<float*>(take(tiles * 4));
  s.Z = reinterpret_cast<float*>(take(tiles * 4));
  s.bytes = off;
  return s;
}

DeltaWork delta_work_view(void* base, const DeltaArgs& a) {
  DeltaWork w;
  size_t off = 0;
  auto take = [&](size_t values) {
    float* p = reinterpret_cast<float*>(static_cast<char*>(base) + off);
    off += align256(4 * values);
    return p;
  };
  const size_t tiles = (size_t)a.B * a.Hv * a.NC * kTile2;
  w.E = take(tiles);
  w.F = take(tiles);
  w.dS = take(tiles);
  w.dZ = take(tiles);
  w.dqh = a.H != a.Hq ? take((size_t)a.B * a.H * a.N * 64) : nullptr;
  w.dkh = a.Hv != a.Hk ? take((size_t)a.B * a.Hv * a.N * 64) : nullptr;
  w.bytes = off;
  return w;
}

template <typename T>
void launch_delta_forward(const DeltaArgs& a, const float* state, void* out, float* final_state, void* saved,
                          hipStream_t st, const Timer& timed) {
  const int U = a.B * a.Hv;
  const DeltaSaved s = delta_saved_view(saved, U, a.NC);
  timed("k_delta_solve", st, [&] { hipLaunchKernelGGL(k_delta_solve<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, s.T); });
  timed("k_delta_scan", st, [&] {
    hipLaunchKernelGGL(k_delta_scan<T>, dim3(U), dim3(kThr), 0, st, a, s.T, state, s.S, s.Z, final_state);
  });
  timed("k_delta_out", st, [&] {
    hipLaunchKernelGGL(k_delta_out<T>, dim3(a.NC * a.B * a.H), dim3(kThr), 0, st, a, s.S, s.Z, static_cast<T*>(out));
  });
}

template <typename T>
void launch_delta_backward(const DeltaArgs& a, const void* saved, const void* dout, const float* dfinal, void* dq,
                           void* dk, void* dv, float* dg, void* dbeta, float* dstate, void* work, hipStream_t st,
                           const Timer& timed) {
  const int U = a.B * a.Hv;
  const DeltaSaved s = delta_saved_view(const_cast<void*>(saved), U, a.NC);
  const DeltaWork w = delta_work_view(work, a);
  const T* od = static_cast<const T*>(dout);
  timed("k_delta_bwd_local", st, [&] {
    hipLaunchKernelGGL(k_delta_bwd_local<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, od, w.E, w.F);
  });
  timed("k_delta_bwd_scan", st, [&] {
    hipLaunchKernelGGL(k_delta_bwd_scan<T>, dim3(U), dim3(kThr), 0, st, a, s.T, dfinal, w.E, w.F, w.dS, w.dZ, dstate);
  });
  timed("k_delta_bwd_out", st, [&] {
    hipLaunchKernelGGL(k_delta_bwd_out<T>, dim3(a.NC * U), dim3(kThr), 0, st, a, od, s.S, s.Z, w.E, w.dS, w.dZ,
                       static_cast<T*>(dq), w.dqh, static_cast<T*>(dk), w.dkh, static_cast<T*>(dv), dg, dbeta);
  });
  auto sum = [&](const float* src, void* dst, int heads, int each) {
    const int64_t head = (int64_t)a.N * 64, total = (int64_t)a.B * heads * head;
    timed("k_delta_sum_heads", st, [&] {
      hipLaunchKernelGGL(k_delta_sum_heads<T>, dim3((unsigned)((total / 4 + kThr - 1) / kThr)), dim3(kThr), 0, st, src,
                         static_cast<T*>(dst), each, head, total);
    });
  };
  if (w.dqh) sum(w.dqh, dq, a.Hq, a.H / a.Hq);
  if (w.dkh) sum(w.dkh, dk, a.Hk, a.Hv / a.Hk);
}

template void launch_delta_forward<float>(const DeltaArgs&, const float*, void*, float*, void*, hipStream_t,
                                          const Timer&);
template void launch_delta_forward<uint16_t>(const DeltaArgs&, const float*, void*, float*, void*, hipStream_t,
                                             const Timer&);
template void launch_delta_backward<float>(const DeltaArgs&, const void*, const void*, const float*, void*, void*,
                                           void*, float*, void*, float*, void*, hipStream_t, const Timer&);
template void launch_delta_backward<uint16_t>(const DeltaArgs&, const void*, const void*, const float*, void*, void*,
                                              void*, float*, void*, float*, void*, hipStream_t, const Timer&);

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
