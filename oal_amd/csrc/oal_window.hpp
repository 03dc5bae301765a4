// Arguments and launches of the windowed attention kernels (oal_window.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oal_delta.hpp"

namespace oal {

// Query i of Nq has position off + i, off = Nk - Nq; it sees keys j <= off + i with
// off + i - j < window or j < sinks.
struct WindowArgs {
  Strided q, k, v;  // rows of D, D and DV values
  int B, Hq, Hk, Nq, Nk, D, DV, window, sinks;
  float scale;
};

// How the key side of the backward is cut: `splits` parts of each block of keys' steps (a
// step: one query head and 64 queries), `chunks` of the steps over which the first keys are seen from afar.
struct WindowPlan {
  int splits, chunks, sink_rows, sink_blocks;
};
// keys: of a block, 128 for bf16 and 64 for the other types
WindowPlan window_plan(int B, int Hq, int Hk, int Nq, int Nk, int window, int sinks, int keys);

struct WindowWork {
  float* delta;   // [B][Hq][Nq] sum of dout * out
  float* part;    // [2][splits][B][Hk][Nk][64] dk and dv of each part
  float* far;     // [2][chunks][B][Hk][sink_rows][64]
  size_t bytes;
};
WindowWork window_work_view(void* base, const WindowArgs& a, const WindowPlan& p);

// lse [B][Hq][Nq]: log2 of each row's sum of exponentials
template <typename T>
void launch_window_forward(const WindowArgs& a, void* out, float* lse, hipStream_t st, const Timer& timed);
template <typename T>
void launch_window_backward(const WindowArgs& a, const void* out, const float* lse, const void* dout, void* dq,
                            void* dk, void* dv, void* work, hipStream_t st, const Timer& timed);

struct WindowStepArgs {
  Strided q, k, v;          // one row per head: the token's
  Strided kc, vc;           // caches [B][Hk][sinks + window][D], rows of D values at stride n
  const int64_t* position;  // [B] tokens before this one; negative: no token here
  int B, Hq, Hk, D, DV, window, sinks, splits, span;
  float scale;
  void* out;    // [B][Hq][DV]
  float* part;  // [splits][B][Hq][DV + 2] (splits > 1)
};
// Slots per block and blocks per head group: from the cache's size and how many head groups fill the chip, so
// the same sequence may be summed in other pieces in another batch.
void window_step_plan(int B, int Hq, int Hk, int64_t slots, int* splits, int* span);
// kind: 0 float32, 1 bfloat16, 2 float16
void launch_window_step(int kind, const WindowStepArgs& a, hipStream_t st, const Timer& timed);

}  // namespace oal
