// Arguments of the short convolution's kernels (conv.hip).
#pragma once
#include "mixer_common.hpp"

namespace lz {

constexpr int CONV_THREADS = 256, CONV_MAX_TAPS = 4;
// Channels a thread.  Eight in the forward, 16 bytes of bf16 a row (5 x 1021 tokens of 2050
// channels: 15 us, with four 19); four in the backward, where eight leave no registers for
// the batches of rows on their way (8192 tokens x 4096 channels: 44.9 us, with eight 46.0).
constexpr int CONV_FWD_V = 8, CONV_BWD_V = 4;

struct Conv {
  const void* x;
  const float *w, *bias;         // [C, K], [C]
  const void* state_in;          // [B, K - 1, C], the rows before the first
  void* state_out;
  const int* lengths;
  void* y;                       // [B, L, C]
  long long x_b;                 // elements from one sequence to the next
  int x_t;                       // and from one token to the next
  int batch, L, C, act;
  // conv_split: columns (vectors of channels) a workgroup, tokens a run, runs a sequence
  int cols, col_blocks, run, seq_runs, run_blocks;
};

void conv_split(Conv& p, bool backward);
hipError_t launch_conv(const Conv& p, int K, const void* dy, void* dx, float* part, bool is_bf16,
                       bool vec, hipStream_t st);
hipError_t launch_conv_sums(const Conv& p, int K, const float* part, float* dw, float* dbias,
                            hipStream_t st);
hipError_t launch_conv_step(const Conv& p, int K, bool is_bf16, hipStream_t st);

}  // namespace lz
