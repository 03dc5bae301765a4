// Arguments and launches of the gated delta rule's kernels (oal_delta.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oal_internal.hpp"

namespace oal {

// A [B][heads][N][..] tensor with unit stride inside a row; strides in elements.
struct Strided {
  const void* p;
  int64_t b, h, n;
};

struct DeltaArgs {
  Strided q, k, v, g, beta;  // rows of D, D and DV values; g and beta one value
  int B, Hq, Hk, Hv, H, N, NC, D, DV;
  bool beta32;  // beta is float32 whatever the other operands are
  float scale;
};

// What the forward computes per unit u = b Hv + state head and chunk, and the backward reads (G to Z).
struct DeltaSaved {
  float* G;  // [U][NC][5][64] its tokens' decays and betas
  float* T;  // [U][NC][64][64] the chunk's solved triangle
  float* M;  // [U][NC][64][64] its map of the state, S' = M S + D
  float* S;  // [U][NC][64][64] state before the chunk
  float* Z;  // [U][NC][64][64] what each token found missing in its state, unscaled by beta (null: not kept)
  float* D;
  float* scratch;
  size_t bytes;
};
DeltaSaved delta_saved_view(void* base, int U, int NC, bool keep);

struct DeltaWork {
  float* E;   // [U][NC][64][64] gradient of u from the chunk's own outputs
  float* F;   // [U][NC][64][64] gradient of the state before the chunk from its outputs
  float* dS;  // [U][NC][64][64] gradient of the state after the chunk
  float* scratch;
  float* dqh;  // [B][H][N][D] dq of every output head (null: heads are not shared)
  float* dkh;  // [B][Hv][N][D] dk of every state head (null: heads are not shared)
  size_t bytes;
};
DeltaWork delta_work_view(void* base, const DeltaArgs& a);

// keep: for a backward
template <typename T>
void launch_delta_forward(const DeltaArgs& a, const float* state, void* out, float* final_state, void* saved, bool keep,
                          hipStream_t st, const Timer& timed);
// dout [B][H][N][DV]; dfinal [U][D][DV] may be null (no gradient).
template <typename T>
void launch_delta_backward(const DeltaArgs& a, const void* saved, const void* dout, const float* dfinal, void* dq,
                           void* dk, void* dv, float* dg, void* dbeta, float* dstate, void* work, hipStream_t st,
                           const Timer& timed);

// dst [B][heads][head values] of src [B][heads each][head values]: sums over heads that one serves, in order.
template <typename T>
void launch_sum_heads(const float* src, T* dst, int B, int heads, int each, int64_t head, hipStream_t st,
                      const Timer& timed);

struct DeltaStepArgs {
  Strided q, k, v, g, beta;
  int B, Hq, Hk, Hv, H, N, Dk, Dv;
  bool beta32;
  float scale;
  float* state;  // [B][Hv][Dk][Dv]
  void* out;     // [B][H][N][Dv]
};
// kind: 0 float32, 1 bfloat16, 2 float16
void launch_delta_step(int kind, const DeltaStepArgs& a, hipStream_t st, const Timer& timed);

}  // namespace oal
