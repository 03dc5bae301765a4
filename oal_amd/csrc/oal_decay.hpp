// Arguments and launches of the kernels of linear attention with decays (oal_decay.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oal_delta.hpp"
#include "oal_internal.hpp"

namespace oal {

struct DecayArgs {
  Strided q, k, v, g;  // rows of D, D and DV values; g one value (strides of 0 where a head has one for all)
  int B, Hq, Hk, Hv, H, N, NC, D, DV;
  bool per_head;  // g's gradient is one value per head
  float scale;
};

// Chunks are walked in segments of `len`.
struct DecaySegments {
  int count, len;
};

// What the forward computes per unit u = b Hv + state head and chunk, and the backward reads (S).
struct DecaySaved {
  float* S;  // [U][NC][64][64] state before the chunk (null: not kept)
  float* G;  // [U][segments][2] the segment's decay, in two parts (nothing for a single one)
  float* D;  // [U][segments][64][64] what it adds to the state, then the state before it
  size_t bytes;
};
DecaySaved decay_saved_view(void* base, int U, int NC, bool keep);

struct DecayWork {
  float* G;     // [U][segments][2]
  float* dS;    // [U][segments][64][64] gradient of the state after the segment
  float* dqh;   // [B][H][N][D] dq of every output head (null: heads are not shared)
  float* dkh;   // [B][Hv][N][D] dk of every state head (null: heads are not shared)
  double* sum;  // [U][NC] sums of dg over the chunk (null: g is per token)
  size_t bytes;
};
DecayWork decay_work_view(void* base, const DecayArgs& a);

// keep: for a backward
template <typename T>
void launch_decay_forward(const DecayArgs& a, const float* state, void* out, float* final_state, void* saved, bool keep,
                          hipStream_t st, const Timer& timed);
// dout [B][H][N][DV]; dfinal [U][D][DV] may be null (no gradient).
template <typename T>
void launch_decay_backward(const DecayArgs& a, const void* saved, const void* dout, const float* dfinal, void* dq,
                           void* dk, void* dv, float* dg, float* dstate, void* work, hipStream_t st,
                           const Timer& timed);

struct DecayStepArgs {
  Strided q, k, v, g;
  int B, Hq, Hk, Hv, H, N, Dk, Dv;
  float scale;
  float* state;  // [B][Hv][Dk][Dv]
  void* out;     // [B][H][N][Dv]
};
// kind: 0 float32, 1 bfloat16, 2 float16
void launch_decay_step(int kind, const DecayStepArgs& a, hipStream_t st, const Timer& timed);

}  // namespace oal
