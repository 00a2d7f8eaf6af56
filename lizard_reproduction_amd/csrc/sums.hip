// Sums of partial results in a fixed order (mixer_common.hpp): the second launch of the
// mixers' backward passes, which add no floats atomically.
//
// A workgroup takes 64 outputs, a lane each, its waves a run of the parts each; the
// waves' sums meet in LDS and are added in wave order.  Consecutive lanes read
// consecutive floats, so a job is as long as its partial results' bytes take (the scan's dB
// and dC of 8192 tokens x 16 states from 64 blocks of channels, 67 MB: 24 us with dA, dD and
// dbias).
#include "mixer_common.hpp"

namespace lz {

constexpr int SUM_WAVES = 8, SUM_BATCH = 8;

constexpr int SUM_GRID = 1 << 22;   // workgroups; more outputs are taken in rounds

struct SumGrid {
  SumJobs jobs;
  long long blk0[SUM_JOBS + 1];
};

__global__ __launch_bounds__(64 * SUM_WAVES) void sums_kernel(SumGrid g) {
  __shared__ float red[SUM_WAVES][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (long long blk = blockIdx.x; blk < g.blk0[g.jobs.n]; blk += SUM_GRID) {
    int j = 0;
#pragma unroll
    for (int i = 1; i < SUM_JOBS; ++i)
      if (i < g.jobs.n && blk >= g.blk0[i]) j = i;
    const SumJob& q = g.jobs.job[j];
    const long long at = (blk - g.blk0[j]) * 64 + lane;
    const bool in = at < (long long)q.sets * q.rows * q.cols;
    long long row = in ? at / q.cols : 0;
    const int col = in ? (int)(at - row * q.cols) : 0;
    const float* src = q.src + col;
    long long out = col * q.out_col;
    if (q.sets > 1) {
      const long long set = row / q.rows;
      row -= set * q.rows;
      src += set * q.set_stride;
      out += set * q.out_set;
    }
    src += row * q.row_stride;
    out += row * q.out_row;
    const int run = (q.parts + SUM_WAVES - 1) / SUM_WAVES;
    const int end = min(q.parts, (wave + 1) * run);
    float sum = 0.f;
    if (in)
      for (int p = wave * run; p < end; p += SUM_BATCH) {
        float v[SUM_BATCH];
#pragma unroll
        for (int k = 0; k < SUM_BATCH; ++k)
          v[k] = src[(long long)min(p + k, end - 1) * q.part_stride];
#pragma unroll
        for (int k = 0; k < SUM_BATCH; ++k) sum += p + k < end ? v[k] : 0.f;
      }
    red[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && in) {
#pragma unroll
      for (int w = 1; w < SUM_WAVES; ++w) sum += red[w][lane];
      if (q.bf16)
        static_cast<bf16*>(q.dst)[out] = to_bf16(sum);
      else
        static_cast<float*>(q.dst)[out] = sum;
    }
    __syncthreads();
  }
}

hipError_t launch_sums(const SumJobs& jobs, hipStream_t st) {
  SumGrid g = {};
  g.jobs = jobs;
  long long blocks = 0;
  for (int i = 0; i < jobs.n; ++i) {
    const SumJob& q = jobs.job[i];
    g.blk0[i] = blocks;
    blocks += ((long long)q.sets * q.rows * q.cols + 63) / 64;
  }
  g.blk0[jobs.n] = blocks;
  if (!blocks) return hipSuccess;
  const unsigned grid = (unsigned)(blocks < SUM_GRID ? blocks : SUM_GRID);
  hipLaunchKernelGGL(sums_kernel, dim3(grid), dim3(64 * SUM_WAVES), 0, st, g);
  return hipGetLastError();
}

}  // namespace lz
