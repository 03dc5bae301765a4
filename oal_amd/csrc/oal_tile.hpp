// Products of 64 x 64 tiles on the matrix cores whose operands are one to three
// bf16 parts, for the chunked and the windowed attention kernels on gfx950.
//
// A value in three bf16 parts (the value rounded, what that left, what that
// left) carries 24 bits, so products of such parts that leave out only the terms below
// 2^-24 are as exact as fp32, at 3 (one operand a bf16 value as it is), 4 (two operands of two parts)
// to 6 matrix instructions in place of the 16 times slower fp32 ones. bf16 tensors enter as
// one part, fp16 tensors as two, fp32 tensors and intermediate results that have to stay fp32 as three.
//
// An accumulator tile of v_mfma_f32_16x16x32_bf16 holds rows 4 g + i in lane group
// g = lane / 16, and an operand's lane group g holds 8 of the 32 indexes that the
// product sums over. Which 8 does not matter as long as both operands agree, so
// two accumulator tiles (32 rows) are, lane for lane, an operand of a product
// that sums over their rows, in the order
//   slot (g, j) -> row 4 g + j (j < 4), 16 + 4 g + j - 4 (j >= 4),
// and the other operand is read from LDS in that order: chains of products
// pass through registers. "perm" marks that order below.
#pragma once

#include <type_traits>

#include "oal_mfma_common.hpp"

namespace oal {

constexpr int kTileElems = 64 * 64;

template <int NP>
struct Frag {
  bf16x8 p[NP];
};

// Exact parts per value of an element type: 24, 8 and 11 bits.
template <typename T>
inline constexpr int kPartsOf = std::is_same_v<T, float> ? 3 : std::is_same_v<T, _Float16> ? 2 : 1;

template <int NP>
__device__ __forceinline__ Frag<NP> split(const float (&v)[8]) {
  Frag<NP> f;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    f.p[p] = pack8(r);
    if (p + 1 < NP) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] -= static_cast<float>(f.p[p][e]);
    }
  }
  return f;
}

// c += a b of the parts i + j <= LAST, small terms first.
template <int LAST, int NA, int NB>
__device__ __forceinline__ f32x4 mma_parts(const Frag<NA>& a, const Frag<NB>& b, f32x4 c) {
#pragma unroll
  for (int s = LAST; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = s - i;
      if (j >= 0 && j < NB) c = mfma16(a.p[i], b.p[j], c);
    }
  return c;
}
// c += a b without the terms of parts below fp32's last bit: part i is at most 2^-8i of its value, so
// those past i + j = 2. Two operands of two parts have all four terms.
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Frag<NA>& a, const Frag<NB>& b, f32x4 c) {
  return mma_parts<(NA + NB - 2 < 2 ? NA + NB - 2 : 2)>(a, b, c);
}
// The same for a b that was itself cut to two parts: what the cut left is up to 2^-16 of a value, and
// so is the product of the low parts, which is left out too (float16 window, 4 x 2048 tokens,
// forward and backward: 457 us, with it 475).
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma_cut(const Frag<NA>& a, const Frag<NB>& b, f32x4 c) {
  return mma_parts<(NA > NB ? NA : NB) - 1>(a, b, c);
}

// LDS tile: NP parts of 64 rows of 64 bf16. The 16-byte piece c of row r stands at c ^ r % 8:
// reads of one column's pieces over 8 rows, and of rows, meet all banks.
__device__ __forceinline__ int tile_at(int r, int c) { return r * 64 + 8 * ((c >> 3) ^ (r & 7)) + (c & 7); }
template <int NP>
struct alignas(16) Tile {
  __bf16 x[NP * kTileElems];
};

// Operand row r0 + lane % 16, sum indexes 32 t + 8 g + j; its first N parts (0: all).
template <int N = 0, int NP>
__device__ __forceinline__ Frag<(N ? N : NP)> row_frag(const Tile<NP>& s, int r0, int t, int lane) {
  Frag<(N ? N : NP)> f;
  const __bf16* p = s.x + tile_at(r0 + (lane & 15), 32 * t + 8 * (lane >> 4));
#pragma unroll
  for (int e = 0; e < (N ? N : NP); ++e) f.p[e] = *reinterpret_cast<const bf16x8*>(p + e * kTileElems);
  return f;
}
// The same row with the sum indexes in perm order.
template <int N = 0, int NP>
__device__ __forceinline__ Frag<(N ? N : NP)> row_frag_perm(const Tile<NP>& s, int r0, int t, int lane) {
  Frag<(N ? N : NP)> f;
  const int r = r0 + (lane & 15), c = 32 * t + 4 * (lane >> 4);
  const __bf16 *p = s.x + tile_at(r, c), *q = s.x + tile_at(r, c + 16);
#pragma unroll
  for (int e = 0; e < (N ? N : NP); ++e) {
    const bf16x4 lo = *reinterpret_cast<const bf16x4*>(p + e * kTileElems);
    const bf16x4 hi = *reinterpret_cast<const bf16x4*>(q + e * kTileElems);
    f.p[e] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// Transposed read: operand row c0 + lane % 16 is a column of the tile, the sum
// indexes are its rows. ds_read_b64_tr_b16 hands lane i of a 16-lane group column i
// of the 4 x 16 block whose row j lanes 4 j .. 4 j + 3 address.
__device__ __forceinline__ bf16x8 tr_rows(const __bf16* lo_row, const __bf16* hi_row) {
  typedef __attribute__((address_space(3))) trv4 lds_trv4;
  const trv4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_trv4*)(lo_row));
  const trv4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_trv4*)(hi_row));
  typedef short trv8 __attribute__((ext_vector_type(8)));
  const trv8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8, v);
}
template <int N = 0, int NP>
__device__ __forceinline__ Frag<(N ? N : NP)> col_frag_perm(const Tile<NP>& s, int c0, int t, int lane) {
  Frag<(N ? N : NP)> f;
  const int g = lane >> 4, i = lane & 15;
  const __bf16* p = s.x + tile_at(32 * t + 4 * g + (i >> 2), c0 + 4 * (i & 3));
#pragma unroll
  for (int e = 0; e < (N ? N : NP); ++e) f.p[e] = tr_rows(p + e * kTileElems, p + e * kTileElems + 16 * 64);
  return f;
}
template <int N = 0, int NP>
__device__ __forceinline__ Frag<(N ? N : NP)> col_frag(const Tile<NP>& s, int c0, int t, int lane) {
  Frag<(N ? N : NP)> f;
  const int g = lane >> 4, i = lane & 15;
  const int r = 32 * t + 8 * g + (i >> 2), c = c0 + 4 * (i & 3);
  const __bf16 *p = s.x + tile_at(r, c), *q = s.x + tile_at(r + 4, c);
#pragma unroll
  for (int e = 0; e < (N ? N : NP); ++e) f.p[e] = tr_rows(p + e * kTileElems, q + e * kTileElems);
  return f;
}

// Two accumulator tiles as the operand of a sum over their 32 rows (perm order).
template <int NP>
__device__ __forceinline__ Frag<NP> acc_frag(const f32x4& lo, const f32x4& hi) {
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return split<NP>(v);
}

// 8 consecutive values of a row as floats, 16-byte aligned.
__device__ __forceinline__ void load_row8(float (&x)[8], const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load_row8(float (&x)[8], const uint16_t* p) {
  const bf16x8 v = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(v[e]);
}
__device__ __forceinline__ void load_row8(float (&x)[8], const _Float16* p) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  const f16x8 v = *reinterpret_cast<const f16x8*>(p);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = static_cast<float>(v[e]);
}

// Four consecutive values of a row, aligned to their size.
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4*>(p); }
__device__ __forceinline__ f32x4 load4(const uint16_t* p) {
  const bf16x4 v = *reinterpret_cast<const bf16x4*>(p);
  return __builtin_convertvector(v, f32x4);
}
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 load4(const _Float16* p) {
  return __builtin_convertvector(*reinterpret_cast<const f16x4*>(p), f32x4);
}
__device__ __forceinline__ void store4(float* p, const f32x4& x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void store4(uint16_t* p, const f32x4& x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
}
__device__ __forceinline__ void store4(_Float16* p, const f32x4& x) {
  *reinterpret_cast<f16x4*>(p) = __builtin_convertvector(x, f16x4);
}
__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ float get(const uint16_t* p) { return to_f(*p); }
__device__ __forceinline__ float get(const _Float16* p) { return static_cast<float>(*p); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(uint16_t* p, float x) { *p = from_f<uint16_t>(x); }
__device__ __forceinline__ void put(_Float16* p, float x) { *p = static_cast<_Float16>(x); }

// Operand row straight from global memory: 8 values at p (not read unless live: zero then).
template <int NP, typename T>
__device__ __forceinline__ Frag<NP> global_frag(const T* p, bool live) {
  Frag<NP> f;
  if constexpr (NP == 1) {
    static_assert(std::is_same_v<T, uint16_t>, "a bf16 value is one part");
    uint4 v = make_uint4(0, 0, 0, 0);
    if (live) v = *reinterpret_cast<const uint4*>(p);
    f.p[0] = __builtin_bit_cast(bf16x8, v);
  } else {
    float x[8] = {};
    if (live) load_row8(x, p);
    f = split<NP>(x);
  }
  return f;
}

// 64 rows of D values, a multiple of 8 up to 64 (row stride in elements, 16-byte aligned rows), on
// their way to an LDS tile by 256 threads: fetch() has the loads of all that a kernel starts
// with in flight together, store() waits for its own. Rows at and past `live` and columns from D are zero.
template <int NP, typename T>
struct Incoming {
  Frag<1> raw[2];
  float x[2][8];
  __device__ __forceinline__ void fetch(const T* __restrict__ src, int64_t stride, int D, int live, int t) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int r = (t >> 3) + 32 * n, c = 8 * (t & 7);
      const bool in = r < live && c < D;
      const T* p = src + (in ? r * stride + c : 0);
      if constexpr (kPartsOf<T> == 1) {
        raw[n] = global_frag<1>(p, true);
        if (!in) raw[n] = Frag<1>{};
      } else {
        load_row8(x[n], p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[n][e] = in ? x[n][e] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(Tile<NP>& s, int t) const {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      __bf16* p = s.x + tile_at((t >> 3) + 32 * n, 8 * (t & 7));
      if constexpr (kPartsOf<T> == 1) {
        *reinterpret_cast<bf16x8*>(p) = raw[n].p[0];
      } else {
        const Frag<NP> f = split<NP>(x[n]);
#pragma unroll
        for (int e = 0; e < NP; ++e) *reinterpret_cast<bf16x8*>(p + e * kTileElems) = f.p[e];
      }
    }
  }
};

// A thread's wave as a scalar: what depends on it branches once per wave.
__device__ __forceinline__ int wave_of(int t) { return __builtin_amdgcn_readfirstlane(t >> 6); }

// Sum over the four lane groups of a wave (lanes of one column).
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ float group_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}

}  // namespace oal
