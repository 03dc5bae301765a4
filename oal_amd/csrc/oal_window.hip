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
inline Shape block_shape(int R) {
  const int groups = (R + 7) / 8, heads = (R + groups - 1) / groups;
  return {heads, std::max(1, 4 / heads), groups};
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

__device__ __forceinline__ bool sees(const WindowArgs& a, bool far, int i, int j) {
  return far ? j < a.sinks && i - j >= a.window : j <= i && i - j < a.window;
}
// Whether positions i0 .. i1 see any, or all, of keys j0 .. j0 + 63.
__device__ __forceinline__ bool sees_any(const WindowArgs& a, bool far, int i0, int i1, int j0) {
  return far ? j0 < a.sinks && i1 - j0 >= a.window : j0 <= i1 && i0 - (j0 + 63) < a.window;
}
__device__ __forceinline__ bool sees_all(const WindowArgs& a, bool far, int i0, int i1, int j0) {
  return far ? j0 + 63 < a.sinks && i0 - (j0 + 63) >= a.window : j0 + 63 <= i0 && i1 - j0 < a.window;
}

}  // namespace

template <typename T>
__global__ __launch_bounds__(512) void k_window_fwd(WindowArgs a, Shape sh, int qblocks, T* __restrict__ out,
                                                    float* __restrict__ lse) {
  constexpr int NP = kPartsOf<T>, CT = kColTiles<T>;
  __shared__ Tile<NP> K, V;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int R = a.Hq / a.Hk;
  int id = blockIdx.x;
  const int qb = id % qblocks;
  id /= qblocks;
  const int hg = id % sh.groups;
  id /= sh.groups;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int r = hg * sh.heads + w / sh.subs, off = a.Nk - a.Nq;
  const int span = sh.subs * kCols<T>, q0 = qb * span + (w % sh.subs) * kCols<T>;
  const bool works = r < R && q0 < a.Nq;
  const int h = hk * R + (r < R ? r : R - 1);
  const Keys keys(a, off + qb * span, off + min(a.Nq, (qb + 1) * span) - 1);
  const int i0 = off + q0, i1 = off + min(a.Nq, q0 + kCols<T>) - 1;

  Frag<NP> qf[CT][2];
#pragma unroll
  for (int x = 0; x < CT; ++x)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int row = q0 + 16 * x + c;
      const bool live = row < a.Nq;
      qf[x][s] = global_frag<NP>(rows_at<T>(a.q, b, h, live ? row : 0) + 32 * s + 8 * g, live && 32 * s + 8 * g < a.D);
    }
  f32x4 acc[CT][4] = {};
  float top[CT], sum[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) top[x] = kNone, sum[x] = 0.f;
  const float scale = a.scale * kLog2e;

  for (int tile = 0; tile < keys.tiles; ++tile) {
    const int j0 = keys.start(tile);
    const bool far = tile < keys.far;
    __syncthreads();
    const int live = min(64, a.Nk - j0);
    if (t < 256) {
      load_tile<64, 256>(K, rows_at<T>(a.k, b, hk, j0), a.k.n, a.D, live, t);
      load_tile<64, 256>(V, rows_at<T>(a.v, b, hk, j0), a.v.n, a.DV, live, t);
    }
    __syncthreads();
    if (!works || !sees_any(a, far, i0, i1, j0)) continue;
    f32x4 s[CT][4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int x = 0; x < CT; ++x) s[x][m] = f32x4{};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> k = row_frag(K, 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) s[x][m] = mma(k, qf[x][e], s[x][m]);
      }
    }
    const bool all = sees_all(a, far, i0, i1, j0);
    Frag<NP> p[CT][2];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      const int i = i0 + 16 * x + c;
      float most = kNone;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = s[x][m][e] * scale;
          s[x][m][e] = all || sees(a, far, i, j0 + 16 * m + 4 * g + e) ? y : kNone;
          most = fmaxf(most, s[x][m][e]);
        }
      most = fmaxf(top[x], group_max(most));
      const float base = most == kNone ? 0.f : most;
      const float keep = __builtin_amdgcn_exp2f(top[x] - base);
      top[x] = most;
      float part = 0.f;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[x][m][e] = __builtin_amdgcn_exp2f(s[x][m][e] - base);
          part += s[x][m][e];
        }
      sum[x] = sum[x] * keep + part;
#pragma unroll
      for (int m = 0; m < 4; ++m) acc[x][m] *= keep;
      p[x][0] = acc_frag<NP>(s[x][0], s[x][1]);
      p[x][1] = acc_frag<NP>(s[x][2], s[x][3]);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> v = col_frag_perm(V, 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) acc[x][m] = mma(v, p[x][e], acc[x][m]);
      }
  }
  if (!works) return;
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = q0 + 16 * x + c;
    const float all = group_sum(sum[x]), inv = 1.f / all;
    if (row >= a.Nq) continue;
    const size_t at = ((size_t)b * a.Hq + h) * a.Nq + row;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (16 * m + 4 * g < a.DV) store4(out + at * a.DV + 16 * m + 4 * g, acc[x][m] * inv);
    if (g == 0) lse[at] = top[x] + __builtin_amdgcn_logf(all);
  }
}

// dq, and for the other side delta_i = do_i.o_i: the forward's walk again.
template <typename T>
__global__ __launch_bounds__(512) void k_window_dq(WindowArgs a, Shape sh, int qblocks, const T* __restrict__ out,
                                                   const float* __restrict__ lse, const T* __restrict__ dout,
                                                   float* __restrict__ delta, T* __restrict__ dq) {
  constexpr int NP = kPartsOf<T>, CT = kColTiles<T>;
  __shared__ Tile<NP> K, V;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int R = a.Hq / a.Hk;
  int id = blockIdx.x;
  const int qb = id % qblocks;
  id /= qblocks;
  const int hg = id % sh.groups;
  id /= sh.groups;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int r = hg * sh.heads + w / sh.subs, off = a.Nk - a.Nq;
  const int span = sh.subs * kCols<T>, q0 = qb * span + (w % sh.subs) * kCols<T>;
  const bool works = r < R && q0 < a.Nq;
  const int h = hk * R + (r < R ? r : R - 1);
  const Keys keys(a, off + qb * span, off + min(a.Nq, (qb + 1) * span) - 1);
  const int i0 = off + q0, i1 = off + min(a.Nq, q0 + kCols<T>) - 1;

  Frag<NP> qf[CT][2], of[CT][2];
  float base[CT], dot[CT];
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = q0 + 16 * x + c;
    const bool live = works && row < a.Nq;
    const size_t at = ((size_t)b * a.Hq + h) * a.Nq + (live ? row : 0);
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int col = 32 * s + 8 * g;
      qf[x][s] = global_frag<NP>(rows_at<T>(a.q, b, h, live ? row : 0) + col, live && col < a.D);
      of[x][s] = global_frag<NP>(dout + at * a.DV + col, live && col < a.DV);
      float o[8] = {}, d[8] = {};
      if (live && col < a.DV) {
        load_row8(o, out + at * a.DV + col);
        load_row8(d, dout + at * a.DV + col);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) y += o[e] * d[e];
    }
    dot[x] = group_sum(y);
    base[x] = live ? lse[at] : 0.f;
    if (live && g == 0) delta[at] = dot[x];
  }
  f32x4 acc[CT][4] = {};
  const float scale = a.scale * kLog2e;

  for (int tile = 0; tile < keys.tiles; ++tile) {
    const int j0 = keys.start(tile);
    const bool far = tile < keys.far;
    __syncthreads();
    const int live = min(64, a.Nk - j0);
    if (t < 256) {
      load_tile<64, 256>(K, rows_at<T>(a.k, b, hk, j0), a.k.n, a.D, live, t);
      load_tile<64, 256>(V, rows_at<T>(a.v, b, hk, j0), a.v.n, a.DV, live, t);
    }
    __syncthreads();
    if (!works || !sees_any(a, far, i0, i1, j0)) continue;
    f32x4 s[CT][4], d[CT][4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int x = 0; x < CT; ++x) s[x][m] = f32x4{}, d[x][m] = f32x4{};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> k = row_frag(K, 16 * m, e, lane), v = row_frag(V, 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          s[x][m] = mma(k, qf[x][e], s[x][m]);
          d[x][m] = mma(v, of[x][e], d[x][m]);
        }
      }
    }
    const bool all = sees_all(a, far, i0, i1, j0);
    Frag<NP> p[CT][2];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      const int i = i0 + 16 * x + c;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = __builtin_amdgcn_exp2f(s[x][m][e] * scale - base[x]);
          const float z = y * (d[x][m][e] - dot[x]);
          s[x][m][e] = all || sees(a, far, i, j0 + 16 * m + 4 * g + e) ? z : 0.f;
        }
      p[x][0] = acc_frag<NP>(s[x][0], s[x][1]);
      p[x][1] = acc_frag<NP>(s[x][2], s[x][3]);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> k = col_frag_perm(K, 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) acc[x][m] = mma(k, p[x][e], acc[x][m]);
      }
  }
  if (!works) return;
#pragma unroll
  for (int x = 0; x < CT; ++x) {
    const int row = q0 + 16 * x + c;
    if (row >= a.Nq) continue;
    const size_t at = ((size_t)b * a.Hq + h) * a.Nq + row;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (16 * m + 4 * g < a.D) store4(dq + at * a.D + 16 * m + 4 * g, acc[x][m] * a.scale);
  }
}

// dk and dv of 4 waves' keys over a part of the queries that see them. Blocks
// 0 .. near - 1: through the window; the others: first keys seen from afar.
template <typename T>
__global__ __launch_bounds__(256) void k_window_dkv(WindowArgs a, WindowPlan plan, int kblocks, int near,
                                                    const float* __restrict__ lse, const T* __restrict__ dout,
                                                    const float* __restrict__ delta, float* __restrict__ part,
                                                    float* __restrict__ farpart) {
  constexpr int NP = kPartsOf<T>, CT = kColTiles<T>;
  __shared__ Tile<NP> Q, O;
  __shared__ alignas(16) float base[64], dot[64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
  const int R = a.Hq / a.Hk, off = a.Nk - a.Nq;
  const bool far = (int)blockIdx.x >= near;
  const int blocks = far ? plan.sink_blocks : kblocks, parts = far ? plan.chunks : plan.splits;
  const int rows = far ? plan.sink_rows : a.Nk;
  int id = far ? blockIdx.x - near : blockIdx.x;
  const int kb = id % blocks;
  id /= blocks;
  const int piece = id % parts;
  id /= parts;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int jb = kb * 4 * kCols<T>, j0 = jb + w * kCols<T>;
  // positions of the queries that see these keys
  const int last = min(rows, jb + 4 * kCols<T>) - 1;
  const int lo = max(off, far ? jb + a.window : jb);
  const int64_t until = far ? a.Nk - 1 : min((int64_t)a.Nk - 1, (int64_t)last + a.window - 1);
  const int tiles = until >= lo ? (int)(until - lo) / 64 + 1 : 0;
  const int64_t steps = (int64_t)R * tiles;
  const int64_t s0 = steps * piece / parts, s1 = steps * (piece + 1) / parts;

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
  for (int64_t step = s0; step < s1; ++step) {
    const int h = hk * R + (int)(step / tiles), i0 = lo + 64 * (int)(step % tiles);  // position of the tile's first query
    const int live = min(64, a.Nk - i0);
    const size_t at = ((size_t)b * a.Hq + h) * a.Nq + (i0 - off);
    __syncthreads();
    load_tile<64, 256>(Q, rows_at<T>(a.q, b, h, i0 - off), a.q.n, a.D, live, t);
    load_tile<64, 256>(O, dout + at * a.DV, (int64_t)a.DV, a.DV, live, t);
    if (t < 64) {
      base[t] = t < live ? lse[at + t] : 0.f;
      dot[t] = t < live ? delta[at + t] : 0.f;
    }
    __syncthreads();
    if (j0 >= rows) continue;
    const int j1 = j0 + kCols<T> - 1, i1 = i0 + live - 1;
    // none, or all, of the pairs in sight
    if (far ? j0 >= a.sinks || i1 - j0 < a.window : j0 > i1 || i0 - j1 >= a.window) continue;
    const bool all = live == 64 && (far ? j1 < a.sinks && i0 - j1 >= a.window : j1 <= i0 && i1 - j0 < a.window);
    f32x4 s[CT][4], d[CT][4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int x = 0; x < CT; ++x) s[x][m] = f32x4{}, d[x][m] = f32x4{};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> q = row_frag(Q, 16 * m, e, lane), o = row_frag(O, 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          s[x][m] = mma(q, kf[x][e], s[x][m]);
          d[x][m] = mma(o, vf[x][e], d[x][m]);
        }
      }
    }
    Frag<NP> p[CT][2], z[CT][2];
#pragma unroll
    for (int x = 0; x < CT; ++x) {
      const int j = j0 + 16 * x + c;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const f32x4 bs = *reinterpret_cast<const f32x4*>(base + 16 * m + 4 * g);
        const f32x4 dt = *reinterpret_cast<const f32x4*>(dot + 16 * m + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = 16 * m + 4 * g + e;
          const float y = __builtin_amdgcn_exp2f(s[x][m][e] * scale - bs[e]);
          const bool seen = all || (row < live && sees(a, far, i0 + row, j));
          s[x][m][e] = seen ? y : 0.f;
          d[x][m][e] = seen ? y * (d[x][m][e] - dt[e]) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[x][e] = acc_frag<NP>(s[x][2 * e], s[x][2 * e + 1]);
        z[x][e] = acc_frag<NP>(d[x][2 * e], d[x][2 * e + 1]);
      }
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const Frag<NP> q = col_frag_perm(Q, 16 * m, e, lane), o = col_frag_perm(O, 16 * m, e, lane);
#pragma unroll
        for (int x = 0; x < CT; ++x) {
          dk[x][m] = mma(q, z[x][e], dk[x][m]);
          dv[x][m] = mma(o, p[x][e], dv[x][m]);
        }
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

// The parts' sums, in order: dk [B][Hk][Nk][D] and dv [B][Hk][Nk][DV].
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
// ---------------------------------------------------------------------------
namespace {

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
  // 32 rows of V per wave; after the walk the waves' sums
  struct alignas(16) Rows {
    __bf16 x[NP * 32 * kTileRow];
  };
  __shared__ Rows V[4];
  __shared__ alignas(16) float acc4[4][16][68];
  __shared__ float top4[4][16], sum4[4][16];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, g = lane >> 4, c = lane & 15;
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
  f32x4 acc[4] = {};
  float top = kNone, sum = 0.f;
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
    float part = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[m][e] = __builtin_amdgcn_exp2f(s[m][e] - base);
        part += s[m][e];
      }
    sum = sum * keep + part;
    const Frag<NP> p = acc_frag<NP>(s[0], s[1]);
    // a wave's LDS accesses are in order: its own rows need no barrier
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const Frag<NP> f = frag_of<T>(vr[x]);
#pragma unroll
      for (int e = 0; e < NP; ++e)
        *reinterpret_cast<bf16x8*>(V[w].x + e * 32 * kTileRow + (8 * x + (lane >> 3)) * kTileRow + 8 * (lane & 7)) = f.p[e];
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
      acc[m] = mma(v, p, acc[m]);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
  sum = group_sum(sum);
  if (g == 0) top4[w][c] = top, sum4[w][c] = sum;
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

template <typename T>
__global__ __launch_bounds__(64) void k_window_step_join(WindowStepArgs a) {
  const size_t head = blockIdx.x, heads = (size_t)a.B * a.Hq;
  const int d = threadIdx.x, width = a.DV + 2;
  if (d >= a.DV) return;
  float most = kNone;
  for (int p = 0; p < a.splits; ++p) most = fmaxf(most, a.part[(p * heads + head) * width + a.DV]);
  float y = 0.f, l = 0.f;
  for (int p = 0; p < a.splits; ++p) {
    const float* x = a.part + (p * heads + head) * width;
    const float f = x[a.DV] == kNone ? 0.f : __builtin_amdgcn_exp2f(x[a.DV] - most);
    y += f * x[d];
    l += f * x[a.DV + 1];
  }
  put(static_cast<T*>(a.out) + head * a.DV + d, a.position[head / a.Hq] < 0 ? 0.f : y / l);
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------
WindowPlan window_plan(int B, int Hq, int Hk, int Nq, int Nk, int window, int sinks, int keys) {
  WindowPlan p;
  const int R = Hq / Hk;
  const int64_t blocks = (int64_t)B * Hk * ((Nk + keys - 1) / keys);
  // parts until every CU has a few blocks
  p.splits = (int)std::clamp<int64_t>((768 + blocks - 1) / blocks, 1, R);
  p.sink_rows = std::max(0, std::min(sinks, Nk - window));
  p.sink_blocks = (p.sink_rows + keys - 1) / keys;
  const int64_t steps = (int64_t)R * ((std::min(Nq, Nk - std::min(window, Nk)) + 63) / 64);
  p.chunks = p.sink_rows ? (int)std::clamp<int64_t>(steps / 8, 1, 64) : 0;
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
  const Shape sh = block_shape(a.Hq / a.Hk);
  const int qblocks = (a.Nq + sh.subs * kCols<T> - 1) / (sh.subs * kCols<T>);
  // at least the four waves that load the tiles
  const int waves = std::max(4, sh.heads * sh.subs);
  timed("k_window_fwd", st, [&] {
    hipLaunchKernelGGL(k_window_fwd<T>, dim3((unsigned)((int64_t)a.B * a.Hk * sh.groups * qblocks)), dim3(64 * waves), 0,
                       st, a, sh, qblocks, static_cast<T*>(out), lse);
  });
}

template <typename T>
void launch_window_backward(const WindowArgs& a, const void* out, const float* lse, const void* dout, void* dq,
                            void* dk, void* dv, void* work, hipStream_t st, const Timer& timed) {
  const Shape sh = block_shape(a.Hq / a.Hk);
  const int qblocks = (a.Nq + sh.subs * kCols<T> - 1) / (sh.subs * kCols<T>);
  const int waves = std::max(4, sh.heads * sh.subs);
  const WindowPlan plan = window_plan(a.B, a.Hq, a.Hk, a.Nq, a.Nk, a.window, a.sinks, 4 * kCols<T>);
  const WindowWork w = window_work_view(work, a, plan);
  timed("k_window_dq", st, [&] {
    hipLaunchKernelGGL(k_window_dq<T>, dim3((unsigned)((int64_t)a.B * a.Hk * sh.groups * qblocks)), dim3(64 * waves), 0,
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
  // blocks of 128 slots and more, until every CU has two
  const int64_t groups = (int64_t)B * Hk * ((Hq / Hk + 15) / 16);
  const int64_t want = std::clamp<int64_t>(512 / std::max<int64_t>(1, groups), 1, (slots + 127) / 128);
  const int64_t each = ((slots + want - 1) / want + 127) / 128 * 128;
  *span = (int)each;
  *splits = (int)((slots + each - 1) / each);
}

void launch_window_step(int kind, const WindowStepArgs& a, hipStream_t st, const Timer& timed) {
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    const int groups = (a.Hq / a.Hk + 15) / 16;
    timed("k_window_step", st, [&] {
      hipLaunchKernelGGL(k_window_step<T>, dim3((unsigned)((int64_t)a.B * a.Hk * groups * a.splits)), dim3(256), 0, st, a);
    });
    if (a.splits > 1)
      timed("k_window_step_join", st,
            [&] { hipLaunchKernelGGL(k_window_step_join<T>, dim3(a.B * a.Hq), dim3(64), 0, st, a); });
  };
  if (kind == 0)
    launch(0.f);
  else if (kind == 1)
    launch(uint16_t{});
  else
    launch(_Float16{});
}

}  // namespace oal
