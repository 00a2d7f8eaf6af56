// Sums of partial results in a fixed order (mixer_common.hpp): the second launch of the
// mixers' backward passes, which add no floats atomically.
//
// A workgroup takes 64 outputs, a lane each, its waves a run of the parts each; the
// waves' sums meet in LDS and are added in wave order.  Consecutive lanes read
// consecutive floats, so a job is as long as its partial results' bytes take.
#include "mixer_common.hpp"

namespace lz {

constexpr int SUM_WAVES = 8, SUM_BATCH = 8;

struct SumGrid {
  SumJobs jobs;
  int blk0[SUM_JOBS + 1];
};

__global__ __launch_bounds__(64 * SUM_WAVES) void sums_kernel(SumGrid g) {
  __shared__ float red[SUM_WAVES][64];
  int j = 0;
#pragma unroll
  for (int i = 1; i < SUM_JOBS; ++i)
    if (i < g.jobs.n && (int)blockIdx.x >= g.blk0[i]) j = i;
  const SumJob& q = g.jobs.job[j];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long at = (long long)((int)blockIdx.x - g.blk0[j]) * 64 + lane;
  const bool in = at < (long long)q.rows * q.cols;
  const long long row = in ? at / q.cols : 0;
  const int col = in ? (int)(at - row * q.cols) : 0;
  const float* src = q.src + row * q.row_stride + col;
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
  if (wave || !in) return;
#pragma unroll
  for (int w = 1; w < SUM_WAVES; ++w) sum += red[w][lane];
  const long long out = row * q.out_row + col * q.out_col;
  if (q.bf16)
    static_cast<bf16*>(q.dst)[out] = to_bf16(sum);
  else
    static_cast<float*>(q.dst)[out] = sum;
}

hipError_t launch_sums(const SumJobs& jobs, hipStream_t st) {
  SumGrid g = {};
  g.jobs = jobs;
  long long blocks = 0;
  for (int i = 0; i < jobs.n; ++i) {
    g.blk0[i] = (int)blocks;
    blocks += ((long long)jobs.job[i].rows * jobs.job[i].cols + 63) / 64;
  }
  if (!blocks) return hipSuccess;
  if (blocks >= (1LL << 31)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(sums_kernel, dim3((unsigned)blocks), dim3(64 * SUM_WAVES), 0, st, g);
  return hipGetLastError();
}

}  // namespace lz
