// Causal softmax attention over a sliding window and a few first tokens that stay
// visible, for gfx950: forward, backward, and single tokens over a ring cache.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i)  over j <= i with i - j < window or j < sinks
//   dv_j = sum_i p_ij do_i,  ds_ij = scale p_ij (do_i.v_j - do_i.o_i),  dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i
//
// One pass over the keys with the running maximum and sum of each row. All score tiles
// are formed with what a wave owns (32 queries, or 32 keys for dk and dv) as
// columns, so that the scores and their gradients are operands of the next product
// where they stand (oal_tile.hpp). The keys that a block of queries sees are two
// ranges: the first keys that its window has left behind, and the window.
//
// Scores, maxima, sums and results are fp32. For bf16 tensors the weights p are
// rounded to bf16 where they meet v or do: by at most half a step (2^-8 of a weight), with
// independent signs over a row, beside the result's own rounding. The sums of the weights
// are of the rounded ones, so they still average. ds takes two parts (16 bits): it has
// both signs, and what cancels would leave the roundings (with one part dq and dk were off
// by 2.5e-3 to 2.7e-3 of their norm in place of 1.8e-3 to 2.1e-3).
//
// Figures at the kernels: bfloat16, 4 x 4096 tokens of 14 query and 2 KV heads, window 1024.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "oal_common.hpp"
#include "oal_tile.hpp"
#include "oal_window.hpp"

namespace oal {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -__builtin_inff();
constexpr float kFloor = -3.402823466e38f;  // before the first maximum: no finite score is below it

template <typename T>
__device__ __forceinline__ const T* rows_at(const Strided& s, int b, int h, int64_t row) {
  return static_cast<const T*>(s.p) + b * s.b + h * s.h + row * s.n;
}

// Columns per wave: two tiles of 16 share each operand read from LDS; with several parts
// per value the registers hold one.
template <typename T>
constexpr int kColTiles = kPartsOf<T> > 1 ? 1 : 2;
template <typename T>
constexpr int kCols = 16 * kColTiles<T>;

// A block's waves: `heads` query heads of one KV head, `subs` tiles of queries each.
struct Shape {
  int heads, subs, groups;
};
inline Shape block_shape(int R, int most) {
  const int groups = (R + most - 1) / most, heads = (R + groups - 1) / groups;
  return {heads, std::max(1, 4 / heads), groups};
}

// The chip's 8 dies take workgroups in turn and each has its own L2: item of
// workgroup id such that every die works on a contiguous range of items.
__device__ __forceinline__ int die_item(int id, int total) {
  const int each = total / 8, more = total % 8, die = id & 7;
  return die * each + min(die, more) + (id >> 3);
}

struct Keys {
  int far, tiles, lo;  // tiles of first keys, all tiles, start of the window's keys
  __device__ Keys(const WindowArgs& a, int first, int last) {
    // positions first .. last of the block's queries
    const int left = min(a.sinks, last - a.window + 1);
    far = left > 0 ? (left + 63) / 64 : 0;
    lo = max(0, first - a.window + 1);
    tiles = far + (last - lo) / 64 + 1;
  }
  __device__ int start(int t) const { return t < far ? 64 * t : lo + 64 * (t - far); }
};

// The pairs of a tile that are seen: distances i - j from `least` on, `count` of them, of
// keys before `keys`.
struct Sight {
  int least;
  unsigned count;
  int keys;
  __device__ Sight(const WindowArgs& a, bool far)
      : least(far ? a.window : 0), count(far ? ~0u >> 1 : a.window), keys(far ? a.sinks : a.Nk) {}
  __device__ bool operator()(int i, int j) const { return ((unsigned)(i - j - least) < count) & (j < keys); }
};
// The largest of 8 results of VALU instructions (no operand is quieted first, as fmaxf does).
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}
__device__ __forceinline__ float largest(const float (&y)[8]) {
  return max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), max3(y[6], y[7], y[7]));
}
template <int NP>
__device__ __forceinline__ Frag<NP> negated(Frag<NP> f) {
#pragma unroll
  for (int e = 0; e < NP; ++e) f.p[e] = -f.p[e];
  return f;
}
// Whether positions i0 .. i1 see any, or all, of keys j0 .. j1.
__device__ __forceinline__ bool sees_any(const WindowArgs& a, bool far, int i0, int i1, int j0, int j1) {
  return far ? j0 < a.sinks && i1 - j0 >= a.window : j0 <= i1 && i0 - j1 < a.window;
}
__device__ __forceinline__ bool sees_all(const WindowArgs& a, bool far, int i0, int i1, int j0, int j1) {
  return far ? j1 < a.sinks && i0 - j1 >= a.window : j1 <= i0 && i1 - j0 < a.window;
}

// 64 rows of a tensor into an LDS tile by a block's 256 threads; bf16 rows go there
// without passing registers, 16 bytes a lane in the order of the lanes. Rows past the last and columns
// past the width repeat others: what they meet is masked or a zero of the other operand.
// Two barriers around it: all waves past their reads before, all rows there behind
// (__syncthreads waits for the copies).
template <int NP, typename T>
__device__ __forceinline__ void bring(Tile<NP>& s, const T* src, int64_t stride, int D, int live, int t) {
  if constexpr (NP == 1) {
    const int lane = t & 63, w = wave_of(t), c = 8 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = 32 * n + 8 * w + (lane >> 3);
      copy16_to_lds(src + (unsigned)(min(r, live - 1) * (int)stride + min(c, D - 8)), s.x + (32 * n + 8 * w) * 64);
    }
  } else {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = (t >> 3) + 32 * n, c = 8 * (t & 7);
      float x[8];
      load_row8(x, src + (unsigned)(min(r, live - 1) * (int)stride + min(c, D - 8)));
      const Frag<NP> f = split<NP>(x);
#pragma unroll
      for (int e = 0; e < NP; ++e) *reinterpret_cast<bf16x8*>(s.x + e * kTileElems + tile_at(r, c)) = f.p[e];
    }
  }
}

// What a block of the query side works on.
struct Block {
  int b, hk, h, q0, i0, i1, first, last;
  bool works;
};
template <typename T>
__device__ __forceinline__ Block query_block(const WindowArgs& a, const Shape& sh, int qblocks, int w) {
  Block x;
  const int R = a.Hq / a.Hk, off = a.Nk - a.Nq;
  int id = die_item(blockIdx.x, gridDim.x);
  const int qb = id % qblocks;
  id /= qblocks;
  const int hg = id % sh.groups;
  id /= sh.groups;
  x.hk = id % a.Hk, x.b = id / a.Hk;
  const int r = hg * sh.heads + w / sh.subs, span = sh.subs * kCols<T>;
  x.q0 = qb * span + (w % sh.subs) * kCols<T>;
  x.works = w < sh.heads * sh.subs && r < R && x.q0 < a.Nq;
  x.h = x.hk * R + min(r, R - 1);
  x.first = off + qb * span, x.last = off + min(a.Nq, (qb + 1) * span) - 1;
  x.i0 = off + x.q0, x.i1 = off + min(a.Nq, x.q0 + kCols<T>) - 1;
  return x;
}

}  // namespace

// A half tile (32 queries by 32 keys) takes a SIMD 930 cycles (740 in a long sequence): vector
// instructions issue for 573 (504), 16 exponentials of 8 among them, and 18 matrix instructions run
// for 288. Neither unit is full (62 to 68 % and 31 to 39 % busy), and waves wait 37 to 39 % of
// their time: a tile is loaded, waited for and then used. The sums of the weights are a third product, with ones, of
// the weights as the values meet them. A row's maximum is moved only when a score
// exceeds it by 2^8, which float32 sums do not mind: else nothing is rescaled.
// Four waves per SIMD (128 registers). 106 us, 498 TFLOP/s of the two products; one
// sequence of 32768 tokens, window 4096: 619 us, 729 TFLOP/s.
template <typename T>
__global__ __launch_bounds__(256, kPartsOf<T> == 1 ? 4 : 1)
void k_window_fwd(WindowArgs a, Shape sh, int qblocks, T* __restrict__ out, float* __restrict__ lse) {
  constexpr int NP = kPartsOf<T>, CT = kColTiles<T>;
  __shared__ Tile<NP> K, V;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const Block at = query_block<T>(a, sh, qblocks, w);
  const Keys keys(a, at.first, at.last);

  Frag<NP> qf[CT][2];
#pragma unroll
  for (int x = 0; x < CT; ++x)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int row = at.q0 + 16 * x + c;
      const bool live = row < a.Nq;
      const int col = 32 * s + 8 * g;
      qf[x][s] = global_frag<NP>(rows_at<T>(a.q, at.b, at.h, live ? row : 0) + col, live && col < a.D);
      if (a.scale < 0.f) qf[x][s] = negated(qf[x][s]);
    }
  Frag<1> ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones.p[0][e] = static_cast<__bf16>(1.f);
  f32x4 acc[CT][4] = {}, sum[CT] = {};
  float top[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) top[x] = kFloor;
  const float scale = fabsf(a.scale) * kLog2e;

  // 32 keys
  auto half_tile = [&](bool masked, bool far, int jh, int half) {
    // the scores that are hidden become none
    auto hide = [&](float (&y)[8], int x) {
      if (masked) {
        const Sight sees(a, far);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[e] = sees(at.i0 + 16 * x + c, jh + 16 * (e >> 2) + 4 * g + (e & 3)) ? y[e] : kNone;
      }
    };
    f32x4 s[CT][2] = {};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> k = row_frag(K, 32 * half + 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) s[x][m] = mma(k, qf[x][e], s[x][m]);
      }
    float y[CT][8], most[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[x][e] = __builtin_fmaf(s[x][e >> 2][e & 3], scale, -top[x]);
      hide(y[x], x);
      most[x] = largest(y[x]);
    }
    if (__any(max3(most[0], most[CT - 1], most[0]) > 8.f)) {
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        // from the stand-in of the start the differences are not exact
#pragma unroll
        for (int e = 0; e < 8; ++e) y[x][e] = s[x][e >> 2][e & 3] * scale;
        hide(y[x], x);
        const float peak = fmaxf(top[x], group_max(largest(y[x]))), less = __builtin_amdgcn_exp2f(top[x] - peak);
        top[x] = peak;
        sum[x] *= less;
#pragma unroll
        for (int m = 0; m < 4; ++m) acc[x][m] *= less;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[x][e] -= peak;
      }
    }
    Frag<NP> p[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[x][e] = __builtin_amdgcn_exp2f(y[x][e]);
      p[x] = split<NP>(y[x]);
      sum[x] = mma(ones, p[x], sum[x]);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const Frag<NP> v = col_frag_perm(V, 16 * m, half, lane);
#pragma unroll
      for (int x = 0; x < CT; ++x) acc[x][m] = mma_cut(v, p[x], acc[x][m]);
    }
  };
  for (int tile = 0; tile < keys.tiles; ++tile) {
    const int j0 = keys.start(tile), live = min(64, at.last + 1 - j0);
    const bool far = tile < keys.far;
    if (tile) lds_sync();
    bring(K, rows_at<T>(a.k, at.b, at.hk, j0), a.k.n, a.D, live, t);
    bring(V, rows_at<T>(a.v, at.b, at.hk, j0), a.v.n, a.DV, live, t);
    __syncthreads();
    if (!at.works) continue;
#pragma nounroll
    for (int half = 0; half < 2; ++half) {
      const int jh = j0 + 32 * half;
      if (!sees_any(a, far, at.i0, at.i1, jh, jh + 31)) continue;
      half_tile(!sees_all(a, far, at.i0, at.i1, jh, jh + 31), far, jh, half);
    }
  }
  if (!at.works) return;
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = at.q0 + 16 * x + c;
    if (row >= a.Nq) continue;
    const float all = sum[x][0], inv = 1.f / all;
    const size_t to = ((size_t)at.b * a.Hq + at.h) * a.Nq + row;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (16 * m + 4 * g < a.DV) store4(out + to * a.DV + 16 * m + 4 * g, acc[x][m] * inv);
    if (g == 0) lse[to] = top[x] + __builtin_amdgcn_logf(all);
  }
}

// dq, and for the other side delta_i = do_i.o_i: the forward's walk again. Matrix cores 36 %
// busy, vector units 58 %, waves waiting 38 %, as in the forward. 155 us, 509 TFLOP/s (135 us with ds in one part).
template <typename T>
__global__ __launch_bounds__(256, kPartsOf<T> == 1 ? 3 : 1)
void k_window_dq(WindowArgs a, Shape sh, int qblocks, const T* __restrict__ out, const float* __restrict__ lse,
                 const T* __restrict__ dout, float* __restrict__ delta, T* __restrict__ dq) {
  constexpr int NP = kPartsOf<T>, NS = NP == 1 ? 2 : NP, CT = kColTiles<T>;
  __shared__ Tile<NP> K, V;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const Block at = query_block<T>(a, sh, qblocks, w);
  const Keys keys(a, at.first, at.last);

  Frag<NP> qf[CT][2], of[CT][2];
  float base[CT], dot[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = at.q0 + 16 * x + c;
    const bool live = at.works && row < a.Nq;
    const size_t from = ((size_t)at.b * a.Hq + at.h) * a.Nq + (live ? row : 0);
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int col = 32 * s + 8 * g;
      qf[x][s] = global_frag<NP>(rows_at<T>(a.q, at.b, at.h, live ? row : 0) + col, live && col < a.D);
      of[x][s] = global_frag<NP>(dout + from * a.DV + col, live && col < a.DV);
      float o[8] = {}, d[8] = {};
      if (live && col < a.DV) {
        load_row8(o, out + from * a.DV + col);
        load_row8(d, dout + from * a.DV + col);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) y += o[e] * d[e];
    }
    dot[x] = group_sum(y);
    base[x] = live ? lse[from] : 0.f;
    if (live && g == 0) delta[from] = dot[x];
  }
  f32x4 acc[CT][4] = {};
  const float scale = a.scale * kLog2e;

  auto half_tile = [&](bool masked, bool far, int jh, int half) {
    f32x4 s[CT][2], d[CT][2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        s[x][m] = f32x4{};
        d[x][m] = f32x4{-dot[x], -dot[x], -dot[x], -dot[x]};
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> k = row_frag(K, 32 * half + 16 * m, e, lane), v = row_frag(V, 32 * half + 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          s[x][m] = mma(k, qf[x][e], s[x][m]);
          d[x][m] = mma(v, of[x][e], d[x][m]);
        }
      }
    }
    Frag<NS> p[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        y[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e >> 2][e & 3], scale, -base[x])) * d[x][e >> 2][e & 3];
      if (masked) {
        const Sight sees(a, far);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[e] = sees(at.i0 + 16 * x + c, jh + 16 * (e >> 2) + 4 * g + (e & 3)) ? y[e] : 0.f;
      }
      p[x] = split<NS>(y);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const Frag<NP> k = col_frag_perm(K, 16 * m, half, lane);
#pragma unroll
      for (int x = 0; x < CT; ++x) acc[x][m] = mma_cut(k, p[x], acc[x][m]);
    }
  };
  for (int tile = 0; tile < keys.tiles; ++tile) {
    const int j0 = keys.start(tile), live = min(64, at.last + 1 - j0);
    const bool far = tile < keys.far;
    if (tile) lds_sync();
    bring(K, rows_at<T>(a.k, at.b, at.hk, j0), a.k.n, a.D, live, t);
    bring(V, rows_at<T>(a.v, at.b, at.hk, j0), a.v.n, a.DV, live, t);
    __syncthreads();
    if (!at.works) continue;
#pragma nounroll
    for (int half = 0; half < 2; ++half) {
      const int jh = j0 + 32 * half;
      if (!sees_any(a, far, at.i0, at.i1, jh, jh + 31)) continue;
      half_tile(!sees_all(a, far, at.i0, at.i1, jh, jh + 31), far, jh, half);
    }
  }
  if (!at.works) return;
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = at.q0 + 16 * x + c;
    if (row >= a.Nq) continue;
    const size_t to = ((size_t)at.b * a.Hq + at.h) * a.Nq + row;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (16 * m + 4 * g < a.D) store4(dq + to * a.D + 16 * m + 4 * g, acc[x][m] * a.scale);
  }
}

// dk and dv of 4 waves' keys over a part of the queries that see them. Blocks
// 0 .. near - 1: through the window; the others: first keys seen from afar. A block's keys
// stay in registers while the queries of all its heads pass, so heads that share keys are
// summed there; parts of them where that leaves CUs empty, summed by k_window_sum in
// order. 185 us, 570 TFLOP/s of the four products (154 us with ds in one part). Three waves per
// SIMD cost bf16 7 spilled registers, loaded again in the loop over steps; two, which hold all, take
// 198 us. Matrix cores 37 % busy, vector units 52 %, waves waiting 43 %.
template <typename T>
__global__ __launch_bounds__(256, kPartsOf<T> == 1 ? 3 : 1)
void k_window_dkv(WindowArgs a, WindowPlan plan, int kblocks, int near, const float* __restrict__ lse,
                  const T* __restrict__ dout, const float* __restrict__ delta, float* __restrict__ part,
                  float* __restrict__ farpart) {
  constexpr int NP = kPartsOf<T>, NS = NP == 1 ? 2 : NP, CT = kColTiles<T>, kKeys = 4 * kCols<T>;
  __shared__ Tile<NP> Q, O;
  __shared__ alignas(16) float base[64], dot[64];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int R = a.Hq / a.Hk, off = a.Nk - a.Nq;
  const bool far = (int)blockIdx.x >= near;
  const int blocks = far ? plan.sink_blocks : kblocks, parts = far ? plan.chunks : plan.splits;
  const int rows = far ? plan.sink_rows : a.Nk;
  int id = far ? blockIdx.x - near : die_item(blockIdx.x, near);
  const int kb = id % blocks;
  id /= blocks;
  const int piece = id % parts;
  id /= parts;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int jb = kb * kKeys, j0 = jb + w * kCols<T>, j1 = j0 + kCols<T> - 1;
  // positions of the queries that see these keys
  const int last = min(rows, jb + kKeys) - 1;
  const int lo = max(off, far ? jb + a.window : jb);
  const int64_t until = far ? a.Nk - 1 : min((int64_t)a.Nk - 1, (int64_t)last + a.window - 1);
  const int tiles = until >= lo ? (int)(until - lo) / 64 + 1 : 0;
  const int64_t steps = (int64_t)R * tiles;
  const int64_t s0 = steps * piece / parts;
  const int count = (int)(steps * (piece + 1) / parts - s0);
  int r = tiles ? (int)(s0 / tiles) : 0, tile = tiles ? (int)(s0 % tiles) : 0;  // of the step
  Frag<NP> kf[CT][2], vf[CT][2];
#pragma unroll
  for (int x = 0; x < CT; ++x)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int row = j0 + 16 * x + c;
      const bool live = row < rows;
      const int col = 32 * s + 8 * g;
      kf[x][s] = global_frag<NP>(rows_at<T>(a.k, b, hk, live ? row : 0) + col, live && col < a.D);
      vf[x][s] = global_frag<NP>(rows_at<T>(a.v, b, hk, live ? row : 0) + col, live && col < a.DV);
    }
  f32x4 dk[CT][4] = {}, dv[CT][4] = {};
  const float scale = a.scale * kLog2e;
  auto half_tile = [&](bool masked, int ih, int half) {
    f32x4 s[CT][2], d[CT][2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const f32x4 dt = *reinterpret_cast<const f32x4*>(dot + 32 * half + 16 * m + 4 * g);
#pragma unroll
      for (int x = 0; x < CT; ++x) s[x][m] = f32x4{}, d[x][m] = dt;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> q = row_frag(Q, 32 * half + 16 * m, e, lane), o = row_frag(O, 32 * half + 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          s[x][m] = mma(q, kf[x][e], s[x][m]);
          d[x][m] = mma(o, vf[x][e], d[x][m]);
        }
      }
    }
    Frag<NP> p[CT];
    Frag<NS> z[CT];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      float y[8], yd[8];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const f32x4 bs = *reinterpret_cast<const f32x4*>(base + 32 * half + 16 * m + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[4 * m + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][m][e], scale, -bs[e]));
          yd[4 * m + e] = y[4 * m + e] * d[x][m][e];
        }
      }
      if (masked) {
        const Sight sees(a, far);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = ih + 16 * (e >> 2) + 4 * g + (e & 3);
          const bool seen = (i < a.Nk) & sees(i, j0 + 16 * x + c);
          y[e] = seen ? y[e] : 0.f;
          yd[e] = seen ? yd[e] : 0.f;
        }
      }
      p[x] = split<NP>(y);
      z[x] = split<NS>(yd);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const Frag<NP> q = col_frag_perm(Q, 16 * m, half, lane), o = col_frag_perm(O, 16 * m, half, lane);
#pragma unroll
      for (int x = 0; x < CT; ++x) {
        dk[x][m] = mma_cut(q, z[x], dk[x][m]);
        dv[x][m] = mma_cut(o, p[x], dv[x][m]);
      }
    }
  };
  for (int step = 0; step < count; ++step) {
    const int h = hk * R + r, i0 = lo + 64 * tile, live = min(64, a.Nk - i0);
    if (++tile == tiles) tile = 0, ++r;
    const size_t at = ((size_t)b * a.Hq + h) * a.Nq + (i0 - off);
    if (step) lds_sync();
    bring(Q, rows_at<T>(a.q, b, h, i0 - off), a.q.n, a.D, live, t);
    bring(O, dout + at * a.DV, a.DV, a.DV, live, t);
    if (t < 64) base[t] = lse[at + min(t, live - 1)];
    if (t >= 64 && t < 128) dot[t - 64] = -delta[at + min(t - 64, live - 1)];
    __syncthreads();
    if (j0 >= rows) continue;
#pragma nounroll
    for (int half = 0; half < 2; ++half) {
      const int ih = i0 + 32 * half, ie = min(a.Nk - 1, ih + 31);
      if (ih >= a.Nk || !sees_any(a, far, ih, ie, j0, j1)) continue;
      half_tile(ie < ih + 31 || !sees_all(a, far, ih, ie, j0, j1), ih, half);
    }
  }
  float* to = far ? farpart : part;
  const size_t half = (size_t)parts * a.B * a.Hk * rows * 64;
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = j0 + 16 * x + c;
    if (row >= rows) continue;
    float* p = to + ((((size_t)piece * a.B + b) * a.Hk + hk) * rows + row) * 64;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      store4(p + 16 * m + 4 * g, dk[x][m] * a.scale);
      store4(p + half + 16 * m + 4 * g, dv[x][m]);
    }
  }
}

// The parts' sums, in order: dk [B][Hk][Nk][D] and dv [B][Hk][Nk][DV]. 21 us.
template <typename T>
__global__ __launch_bounds__(256) void k_window_sum(WindowArgs a, WindowPlan plan, const float* __restrict__ part,
                                                    const float* __restrict__ farpart, T* __restrict__ dk,
                                                    T* __restrict__ dv) {
  const size_t all = (size_t)a.B * a.Hk * a.Nk * 64, x = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (x >= 2 * all) return;
  const bool v = x >= all;
  const size_t y = v ? x - all : x;
  f32x4 s = {};
  for (int p = 0; p < plan.splits; ++p)
    s += *reinterpret_cast<const f32x4*>(part + ((v ? plan.splits : 0) + p) * all + y);
  const size_t bh = y / ((size_t)a.Nk * 64), in = y % ((size_t)a.Nk * 64);
  const size_t rows = (size_t)plan.sink_rows * 64, far = (size_t)a.B * a.Hk * rows;
  if (in < rows)
    for (int p = 0; p < plan.chunks; ++p)
      s += *reinterpret_cast<const f32x4*>(farpart + ((v ? plan.chunks : 0) + p) * far + bh * rows + in);
  const int col = (int)(y & 63), width = v ? a.DV : a.D;
  if (col < width) store4((v ? dv : dk) + (y >> 6) * width + col, s);
}

// ---------------------------------------------------------------------------
// One token over the ring cache: it is written to its slot, and the filled slots
// are just what it sees, in any order. A wave takes 32 slots at a time; its 16
// columns are query heads of one KV head. The slot's row comes from the token itself.
// Bound by the caches' one reading: 128 users of 4100 slots, 2 KV heads, 40 us and the join 4,
// 269 MB at 6.1 TB/s; one user of 1028 slots 5 us and the join 4. float16 takes twice as long (93 us): its
// values are split, with two waves per SIMD.
// ---------------------------------------------------------------------------
namespace {

constexpr int kMostSplits = 512;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

template <typename T>
struct alignas(16) Row8 {
  T v[8];
};
// 8 values of a row of D, D a multiple of 8; zero past D.
template <typename T>
__device__ __forceinline__ Row8<T> row8(const T* p, int d, int D, bool live) {
  Row8<T> r{};
  if (live && d < D) r = *reinterpret_cast<const Row8<T>*>(p + d);
  return r;
}
template <typename T, int NP = kPartsOf<T>>
__device__ __forceinline__ Frag<NP> frag_of(const Row8<T>& r) {
  if constexpr (sizeof(T) == 2 && NP == 1) {
    return Frag<1>{{__builtin_bit_cast(bf16x8, r)}};
  } else {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(r.v[e]);
    return split<NP>(x);
  }
}

}  // namespace

template <typename T>
__global__ __launch_bounds__(256) void k_window_step(WindowStepArgs a) {
  constexpr int NP = kPartsOf<T>;
  // 32 rows of V per wave, 144 bytes each; after the walk the waves' sums
  constexpr int kTileRow = 72;
  struct alignas(16) Rows {
    __bf16 x[NP * 32 * kTileRow];
  };
  __shared__ Rows V[4];
  __shared__ alignas(16) float acc4[4][16][68];
  __shared__ float top4[4][16], sum4[4][16];
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), g = lane >> 4, c = lane & 15;
  const int R = a.Hq / a.Hk, groups = (R + 15) / 16;
  int id = blockIdx.x;
  const int piece = id % a.splits;
  id /= a.splits;
  const int hg = id % groups;
  id /= groups;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int64_t pos = a.position[b], slots = (int64_t)a.sinks + a.window;
  const int count = pos < 0 ? 0 : (int)min(pos + 1, slots);
  const int64_t slot = pos < a.sinks ? pos : a.sinks + (pos - a.sinks) % a.window;
  const int begin = piece * a.span, end = min(count, begin + a.span);
  const T* knew = static_cast<const T*>(a.k.p) + b * a.k.b + hk * a.k.h;
  const T* vnew = static_cast<const T*>(a.v.p) + b * a.v.b + hk * a.v.h;
  T* kc = const_cast<T*>(static_cast<const T*>(a.kc.p)) + b * a.kc.b + hk * a.kc.h;
  T* vc = const_cast<T*>(static_cast<const T*>(a.vc.p)) + b * a.vc.b + hk * a.vc.h;
  if (hg == 0 && pos >= 0 && slot >= begin && slot < begin + a.span) {
    for (int d = t; d < a.D; d += 256) kc[slot * a.kc.n + d] = knew[d];
    for (int d = t; d < a.DV; d += 256) vc[slot * a.vc.n + d] = vnew[d];
  }
  const int r = hg * 16 + c;
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.b + (hk * R + (r < R ? r : 0)) * a.q.h;
  Frag<NP> qf[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) qf[s] = frag_of<T>(row8(q, 32 * s + 8 * g, a.D, r < R));
  Frag<1> ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones.p[0][e] = static_cast<__bf16>(1.f);
  f32x4 acc[4] = {}, sum = {};
  float top = kNone;
  const float scale = a.scale * kLog2e;
  for (int j0 = begin + 32 * w; j0 < end; j0 += 128) {
    Row8<T> kr[2][2], vr[4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int j = j0 + 16 * m + c;
      const T* row = j == slot ? knew : kc + j * a.kc.n;
#pragma unroll
      for (int s = 0; s < 2; ++s) kr[m][s] = row8(row, 32 * s + 8 * g, a.D, j < end);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = j0 + 8 * x + (lane >> 3);
      const T* row = j == slot ? vnew : vc + j * a.vc.n;
      vr[x] = row8(row, 8 * (lane & 7), a.DV, j < end);
    }
    f32x4 s[2] = {};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) s[m] = mma(frag_of<T>(kr[m][e]), qf[e], s[m]);
    float most = kNone;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[m][e] = j0 + 16 * m + 4 * g + e < end ? s[m][e] * scale : kNone;
        most = fmaxf(most, s[m][e]);
      }
    most = fmaxf(top, group_max(most));
    const float base = most == kNone ? 0.f : most;
    const float keep = __builtin_amdgcn_exp2f(top - base);
    top = most;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[m][e] = __builtin_amdgcn_exp2f(s[m][e] - base);
    const Frag<NP> p = acc_frag<NP>(s[0], s[1]);
    // of the weights as the values meet them
    sum *= keep;
    sum = mma(ones, p, sum);
    // a wave's LDS accesses are in order: its own rows need no barrier
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const Frag<NP> f = frag_of<T>(vr[x]);
#pragma unroll
      for (int e = 0; e < NP; ++e)
        *reinterpret_cast<bf16x8*>(V[w].x + (32 * e + 8 * x + (lane >> 3)) * kTileRow + 8 * (lane & 7)) = f.p[e];
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      Frag<NP> v;
      const __bf16* x = V[w].x + (4 * g + (c >> 2)) * kTileRow + 16 * m + 4 * (c & 3);
#pragma unroll
      for (int e = 0; e < NP; ++e) v.p[e] = tr_rows(x + e * 32 * kTileRow, x + e * 32 * kTileRow + 16 * kTileRow);
      acc[m] *= keep;
      acc[m] = mma_cut(v, p, acc[m]);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
  if (g == 0) top4[w][c] = top, sum4[w][c] = sum[0];
#pragma unroll
  for (int m = 0; m < 4; ++m) *reinterpret_cast<f32x4*>(&acc4[w][c][16 * m + 4 * g]) = acc[m];
  __syncthreads();
  for (int x = t; x < 16 * 64; x += 256) {
    const int col = x >> 6, d = x & 63;
    if (hg * 16 + col >= R || d >= a.DV) continue;
    const float most = fmaxf(fmaxf(top4[0][col], top4[1][col]), fmaxf(top4[2][col], top4[3][col]));
    float y = 0.f, l = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = top4[v][col] == kNone ? 0.f : __builtin_amdgcn_exp2f(top4[v][col] - most);
      y += f * acc4[v][col][d];
      l += f * sum4[v][col];
    }
    const size_t head = (size_t)b * a.Hq + hk * R + hg * 16 + col;
    if (a.splits == 1) {
      put(static_cast<T*>(a.out) + head * a.DV + d, pos < 0 ? 0.f : y / l);
    } else {
      float* p = a.part + ((size_t)piece * a.B * a.Hq + head) * (a.DV + 2);
      p[d] = y;
      if (d == 0) p[a.DV] = most, p[a.DV + 1] = l;
    }
  }
}

// The pieces' sums of one head: their weights at once, then a wave per fourth of the pieces.
template <typename T>
__global__ __launch_bounds__(256) void k_window_step_join(WindowStepArgs a) {
  __shared__ float share[kMostSplits], tops[4], sums[4], parts[4][64];
  const size_t head = blockIdx.x, heads = (size_t)a.B * a.Hq;
  const int t = threadIdx.x, lane = t & 63, w = wave_of(t), width = a.DV + 2;
  const float* x = a.part + head * width;
  float most = kNone;
  for (int p = t; p < a.splits; p += 256) {
    share[p] = x[p * heads * width + a.DV];
    most = fmaxf(most, share[p]);
  }
  most = wave_max(most);
  if (lane == 0) tops[w] = most;
  __syncthreads();
  most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  float l = 0.f;
  for (int p = t; p < a.splits; p += 256) {
    const float f = share[p] == kNone ? 0.f : __builtin_amdgcn_exp2f(share[p] - most);
    share[p] = f;
    l += f * x[p * heads * width + a.DV + 1];
  }
  l = wave_sum(l);
  if (lane == 0) sums[w] = l;
  __syncthreads();
  float y = 0.f;
  const int d = min(lane, a.DV - 1);
#pragma unroll 4
  for (int p = w; p < a.splits; p += 4) y += share[p] * x[p * heads * width + d];
  parts[w][lane] = y;
  __syncthreads();
  if (t >= a.DV) return;
  y = (parts[0][t] + parts[1][t]) + (parts[2][t] + parts[3][t]);
  l = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  put(static_cast<T*>(a.out) + head * a.DV + t, a.position[head / a.Hq] < 0 ? 0.f : y / l);
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
WindowPlan window_plan(int B, int Hq, int Hk, int Nq, int Nk, int window, int sinks, int keys) {
  WindowPlan p;
  const int R = Hq / Hk;
  window = std::min(window, Nk), sinks = std::min(sinks, Nk);
  const int64_t blocks = (int64_t)B * Hk * ((Nk + keys - 1) / keys);
  // parts until every CU has three blocks, as many as fit: 4 x 4096 tokens in 3 parts 169 us, in 2 195, in 4 200
  p.splits = (int)std::clamp<int64_t>((768 + blocks - 1) / blocks, 1, R);
  p.sink_rows = std::max(0, std::min(sinks, Nk - window));
  p.sink_blocks = (p.sink_rows + keys - 1) / keys;
  // the first keys' steps in pieces of 8 and more, up to 1024 blocks in all: each piece has sums of its own in memory
  const int64_t steps = (int64_t)R * ((std::min(Nq, Nk - window) + 63) / 64);
  const int64_t sums = (int64_t)B * Hk * p.sink_blocks;
  p.chunks = p.sink_rows ? (int)std::clamp<int64_t>(std::min(steps / 8, 1024 / sums), 1, 64) : 0;
  return p;
}

WindowWork window_work_view(void* base, const WindowArgs& a, const WindowPlan& p) {
  WindowWork w;
  size_t off = 0;
  auto take = [&](size_t values) {
    float* x = reinterpret_cast<float*>(static_cast<char*>(base) + off);
    off += align256(4 * values);
    return x;
  };
  w.delta = take((size_t)a.B * a.Hq * a.Nq);
  w.part = take((size_t)2 * p.splits * a.B * a.Hk * a.Nk * 64);
  w.far = take((size_t)2 * p.chunks * a.B * a.Hk * p.sink_rows * 64);
  w.bytes = off;
  return w;
}

template <typename T>
void launch_window_forward(const WindowArgs& a, void* out, float* lse, hipStream_t st, const Timer& timed) {
  const Shape sh = block_shape(a.Hq / a.Hk, 4);
  const int qblocks = (a.Nq + sh.subs * kCols<T> - 1) / (sh.subs * kCols<T>);
  timed("k_window_fwd", st, [&] {
    hipLaunchKernelGGL(k_window_fwd<T>, dim3((unsigned)((int64_t)a.B * a.Hk * sh.groups * qblocks)), dim3(256), 0,
                       st, a, sh, qblocks, static_cast<T*>(out), lse);
  });
}

template <typename T>
void launch_window_backward(const WindowArgs& a, const void* out, const float* lse, const void* dout, void* dq,
                            void* dk, void* dv, void* work, hipStream_t st, const Timer& timed) {
  const Shape sh = block_shape(a.Hq / a.Hk, 4);
  const int qblocks = (a.Nq + sh.subs * kCols<T> - 1) / (sh.subs * kCols<T>);
  const WindowPlan plan = window_plan(a.B, a.Hq, a.Hk, a.Nq, a.Nk, a.window, a.sinks, 4 * kCols<T>);
  const WindowWork w = window_work_view(work, a, plan);
  timed("k_window_dq", st, [&] {
    hipLaunchKernelGGL(k_window_dq<T>, dim3((unsigned)((int64_t)a.B * a.Hk * sh.groups * qblocks)), dim3(256), 0,
                       st, a, sh, qblocks, static_cast<const T*>(out), lse, static_cast<const T*>(dout), w.delta,
                       static_cast<T*>(dq));
  });
  const int kblocks = (a.Nk + 4 * kCols<T> - 1) / (4 * kCols<T>);
  const int near = a.B * a.Hk * plan.splits * kblocks, far = a.B * a.Hk * plan.chunks * plan.sink_blocks;
  timed("k_window_dkv", st, [&] {
    hipLaunchKernelGGL(k_window_dkv<T>, dim3(near + far), dim3(256), 0, st, a, plan, kblocks, near, lse,
                       static_cast<const T*>(dout), w.delta, w.part, w.far);
  });
  const size_t values = (size_t)2 * a.B * a.Hk * a.Nk * 64;
  timed("k_window_sum", st, [&] {
    hipLaunchKernelGGL(k_window_sum<T>, dim3((unsigned)((values / 4 + 255) / 256)), dim3(256), 0, st, a, plan, w.part,
                       w.far, static_cast<T*>(dk), static_cast<T*>(dv));
  });
}

#define OAL_WINDOW(T)                                                                                              \
  template void launch_window_forward<T>(const WindowArgs&, void*, float*, hipStream_t, const Timer&);             \
  template void launch_window_backward<T>(const WindowArgs&, const void*, const float*, const void*, void*, void*, \
                                          void*, void*, hipStream_t, const Timer&);
OAL_WINDOW(float)
OAL_WINDOW(uint16_t)
OAL_WINDOW(_Float16)
#undef OAL_WINDOW

void window_step_plan(int B, int Hq, int Hk, int64_t slots, int* splits, int* span) {
  // Pieces of 128 slots and more, until every CU has two blocks: one user of 4096 slots 8 us, with
  // pieces of 512 11 us; 96 users 36 us, with one block per CU 47 us. Where each CU has a block
  // already, a short cache is not worth a second launch: 128 users of 1024 slots 17 us, in two pieces 19 us.
  const int64_t groups = (int64_t)B * Hk * ((Hq / Hk + 15) / 16);
  const int64_t pieces = groups >= 256 && slots < 2048 ? 1 : (slots + 127) / 128;
  const int64_t want = std::clamp<int64_t>(kMostSplits / std::max<int64_t>(1, groups), 1, pieces);
  const int64_t each = ((slots + want - 1) / want + 127) / 128 * 128;
  *span = (int)each;
  *splits = (int)((slots + each - 1) / each);
}

void launch_window_step(int kind, const WindowStepArgs& a, hipStream_t st, const Timer& timed) {
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    const int groups = (a.Hq / a.Hk + 15) / 16;
    timed("k_window_step", st, [&] {
      const unsigned blocks = (unsigned)((int64_t)a.B * a.Hk * groups * a.splits);
      hipLaunchKernelGGL(k_window_step<T>, dim3(blocks), dim3(256), 0, st, a);
    });
    if (a.splits > 1)
      timed("k_window_step_join", st,
            [&] { hipLaunchKernelGGL(k_window_step_join<T>, dim3(a.B * a.Hq), dim3(256), 0, st, a); });
  };
  if (kind == 0)
    launch(0.f);
  else if (kind == 1)
    launch(uint16_t{});
  else
    launch(_Float16{});
}

}  // namespace oal
