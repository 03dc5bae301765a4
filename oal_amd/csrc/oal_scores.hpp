// Arguments and launches of the token scores' kernels (oal_scores.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oal_internal.hpp"

namespace oal {

constexpr int kMostTop = 64;

struct ScoreArgs {
  const void* logits;      // [B][N][V], unit stride inside a row
  int64_t b, n;            // strides of the rows, in elements
  const int64_t* tokens;   // [B][N]
  int B, N, V;
  bool entropy;
  int top;
};

struct ScoreOut {
  float* logp;      // [B][N]
  float* entropy;   // [B][N], if asked for
  float* top;       // [B][N][top] log probabilities, if asked for
  int64_t* place;   // [B][N][top] their tokens
  float* saved;     // [B][N][2]: the row's maximum and the sum of exponentials (null: not kept)
};

// Bytes that the parts of rows need before they are joined (0: rows are not cut).
size_t score_work_bytes(const ScoreArgs& a);
template <typename T>
void launch_scores(const ScoreArgs& a, const ScoreOut& out, void* work, hipStream_t st, const Timer& timed);
// dlogits [B][N][V] contiguous; dlog, dentropy [B][N] (null: zero).
template <typename T>
void launch_scores_backward(const ScoreArgs& a, const float* saved, const float* entropy, const float* dlog,
                            const float* dentropy, void* dlogits, hipStream_t st, const Timer& timed);

}  // namespace oal
