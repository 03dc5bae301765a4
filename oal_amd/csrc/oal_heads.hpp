// Arguments and launches of the head norms with rotary embedding (oal_heads.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oal_internal.hpp"

namespace oal {

struct HeadsArgs {
  const void *q, *k, *v;         // projections [B][N][heads D], rows contiguous (backward: q and k)
  int64_t qb, qn, kb, kn, vb, vn;  // their strides, in elements
  const void *qw, *kw;           // weights [D] or [heads][D] (null: none)
  const void *cosine, *sine;     // [table][R]
  const int64_t* position;       // [B][N] (null: 0 .. N - 1)
  int B, N, Hq, Hk, D, R, table;
  bool w32, t32;                 // weights, tables: float32 whatever q is
  bool per_head;                 // a weight for each head
  float eps;
};

// Partial sums of each weight row's gradient that the backward leaves.
int heads_blocks(const HeadsArgs& a);

// hq, hk, hv: [B][heads][N][D].
template <typename T>
void launch_heads_forward(const HeadsArgs& a, void* hq, void* hk, void* hv, hipStream_t st, const Timer& timed);
// Gradients of hq, hk, hv (null: zero) to those of the projections [B][N][heads D] and, with work
// [heads_blocks][per head: Hq + Hk, else 2][D], of the weights (in their type).
template <typename T>
void launch_heads_backward(const HeadsArgs& a, const void* hq, const void* hk, const void* hv, void* dq, void* dk,
                           void* dv, void* dqw, void* dkw, float* work, hipStream_t st, const Timer& timed);

}  // namespace oal
