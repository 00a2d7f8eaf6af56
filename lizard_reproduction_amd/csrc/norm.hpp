// Arguments of the group norm's kernels (norm.hip).
#pragma once
#include "mixer_common.hpp"

namespace lz {

constexpr int NORM_THREADS = 256, NORM_MAX_WIDTH = 8192;

struct Norm {
  const void *x, *gate;          // rows of G groups of W channels
  const float *w, *bias;         // [G W], both or neither
  void* y;                       // [rows, G, W]
  long long x_b, x_t, x_g;       // elements from one sequence, token and group to the next
  long long z_b, z_t, z_g;       // of the gate
  int batch, L, G, W, act;       // act: silu of the result (or of the gate), else neither
  float eps, inv_w;
  // norm_split: threads and vectors a group, groups and rows a workgroup, its grid
  int tpg, vecs, gb, rb, group_blocks, row_blocks;
};

void norm_split(Norm& p, bool backward);
hipError_t launch_norm_fwd(const Norm& p, bool is_bf16, hipStream_t st);
hipError_t launch_norm_bwd(const Norm& p, const void* dy, void* dx, void* dgate, float* part,
                           float* dw, float* dbias, bool is_bf16, hipStream_t st);

}  // namespace lz
