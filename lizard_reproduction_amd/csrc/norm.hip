// Normalisation of groups of channels of each token, with an affine map and an activation:
//
//   n = (x - mean) / sqrt(var + eps) over the group's W channels,  o = n w + b,
//   y = o, silu(o), o gate or o silu(gate)
//
// A group is read once into the registers of as many threads as it has vectors of eight
// channels, its mean and then its squared distances from it summed across them in fp32, so
// the rows' bytes bound it.  A thread keeps its channels, with w and b (backward: the sums
// of dw and db) in registers, and goes through rows; the next row's loads are issued before
// this row is worked on.  Groups may lie apart by any stride (the heads of an attention
// output); y is rows.
//
// Backward, from x again: do = dy act', dn = do w, dx = (dn - mean(dn) - n mean(dn n)) rstd,
// dgate = dy o act'(gate), dw = sum do n, db = sum do.  A workgroup's shares of dw and db go
// to a second launch, which adds them in order.
#include "norm.hpp"

namespace lz {

// Sum over the tpg threads of a group (a power of two; past a wave through LDS)
__device__ __forceinline__ float group_sum(float v, int tpg, float* red) {
  for (int o = 1; o < tpg && o < 64; o *= 2) v += __shfl_xor(v, o);
  if (tpg > 64) {   // uniform
    const int wave = threadIdx.x >> 6, per = tpg >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < per; ++i) v += red[wave / per * per + i];
  }
  return v;
}

struct NormPlace {
  int slot, lane, group;
  bool in;
  __device__ __forceinline__ NormPlace(const Norm& p) {
    lane = threadIdx.x % p.tpg;
    const int i = threadIdx.x / p.tpg;
    slot = i / p.gb;                       // of the rb rows
    group = blockIdx.y * p.gb + i % p.gb;
    in = group < p.G && slot < p.rb;
    if (!in) group = 0;
  }
};

template <typename T, bool VEC, int N>
struct NormRow {
  Cols8<T, VEC> v[N];
  __device__ __forceinline__ void load(const T* base, const Norm& p, int lane) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (j * p.tpg + lane) * 8, left = p.W - e;
      v[j].load(base + (left > 0 ? e : 0), max(left, 1));
    }
  }
};

template <typename T>
__device__ __forceinline__ const T* norm_row(const void* base, long long row, int L, long long sb,
                                             long long stt, long long at) {
  const long long b = (unsigned)row / (unsigned)L;   // rows fit 31 bits
  return (const T*)base + b * sb + (row - b * L) * stt + at;
}

// mean and 1 / sqrt(var + eps) of a group's row
template <typename T, bool VEC, int N>
__device__ __forceinline__ void norm_stats(const NormRow<T, VEC, N>& x, const Norm& p, int lane,
                                           float* red, float& mean, float& rstd) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((j * p.tpg + lane) * 8 + i < p.W) sum += x.v[j].r.at(i);
  mean = group_sum(sum, p.tpg, red) * (1.f / p.W);
  sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((j * p.tpg + lane) * 8 + i < p.W) {
        const float d = x.v[j].r.at(i) - mean;
        sum = fmaf(d, d, sum);
      }
  rstd = 1.f / sqrtf(group_sum(sum, p.tpg, red) * (1.f / p.W) + p.eps);
}

template <typename T, bool VEC, int N>
__global__ __launch_bounds__(NORM_THREADS) void norm_fwd_kernel(Norm p) {
  __shared__ float red[4];
  const NormPlace at(p);
  float w[N][8], bias[N][8];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = (j * p.tpg + at.lane) * 8 + i;
      const size_t ch = (size_t)at.group * p.W + (e < p.W ? e : 0);
      w[j][i] = p.w ? p.w[ch] : 1.f;
      bias[j][i] = p.bias ? p.bias[ch] : 0.f;
    }
  const long long rows = (long long)p.batch * p.L, step = (long long)p.row_blocks * p.rb;
  long long row = (long long)blockIdx.x * p.rb + at.slot;
  NormRow<T, VEC, N> x, z;
  auto load = [&](long long r) {
    r = min(r, rows - 1);
    x.load(norm_row<T>(p.x, r, p.L, p.x_b, p.x_t, at.group * p.x_g), p, at.lane);
    if (p.gate) z.load(norm_row<T>(p.gate, r, p.L, p.z_b, p.z_t, at.group * p.z_g), p, at.lane);
  };
  load(row);
  // every thread makes the same number of rounds: group_sum may hold a barrier
  for (long long first = (long long)blockIdx.x * p.rb; first < rows; first += step, row += step) {
    const NormRow<T, VEC, N> cx = x, cz = z;
    if (first + step < rows) load(row + step);
    float mean, rstd;
    norm_stats(cx, p, at.lane, red, mean, rstd);
    if (!at.in || row >= rows) continue;
    T* y = (T*)p.y + (row * p.G + at.group) * p.W;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (j * p.tpg + at.lane) * 8;
      Cols8<T, VEC> out;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float o = fmaf((cx.v[j].r.at(i) - mean) * rstd, w[j][i], bias[j][i]);
        const float a = p.gate ? cz.v[j].r.at(i) : o;
        if (p.act) o *= p.gate ? a * sigmoid(a) : sigmoid(a);
        else if (p.gate) o *= a;
        out.r.set(i, o);
      }
      if (e < p.W) out.store(y + e, p.W - e);
    }
  }
}

template <typename T, bool VEC, int N>
__global__ __launch_bounds__(NORM_THREADS) void norm_bwd_kernel(Norm p, const void* dy_, void* dx_,
                                                                void* dgate_, float* part) {
  __shared__ float red[4];
  __shared__ float shares[NORM_THREADS][9];
  const NormPlace at(p);
  float w[N][8], bias[N][8], dw[N][8], db[N][8];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = (j * p.tpg + at.lane) * 8 + i;
      const size_t ch = (size_t)at.group * p.W + (e < p.W ? e : 0);
      w[j][i] = e < p.W ? p.w ? p.w[ch] : 1.f : 0.f;
      bias[j][i] = p.bias ? p.bias[ch] : 0.f;
      dw[j][i] = db[j][i] = 0.f;
    }
  const long long rows = (long long)p.batch * p.L, step = (long long)p.row_blocks * p.rb;
  long long row = (long long)blockIdx.x * p.rb + at.slot;
  NormRow<T, VEC, N> x, z, g;
  auto load = [&](long long r) {
    r = min(r, rows - 1);
    x.load(norm_row<T>(p.x, r, p.L, p.x_b, p.x_t, at.group * p.x_g), p, at.lane);
    if (p.gate) z.load(norm_row<T>(p.gate, r, p.L, p.z_b, p.z_t, at.group * p.z_g), p, at.lane);
    g.load((const T*)dy_ + (r * p.G + at.group) * p.W, p, at.lane);
  };
  load(row);
  for (long long first = (long long)blockIdx.x * p.rb; first < rows; first += step, row += step) {
    const NormRow<T, VEC, N> cx = x, cz = z, cg = g;
    if (first + step < rows) load(row + step);
    float mean, rstd;
    norm_stats(cx, p, at.lane, red, mean, rstd);
    const bool have = at.in && row < rows;
    const long long out = (row * p.G + at.group) * p.W;
    float s1 = 0.f, s2 = 0.f, dn[N][8];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (j * p.tpg + at.lane) * 8;
      Cols8<T, VEC> dz;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = have && e + i < p.W;
        const float n = (cx.v[j].r.at(i) - mean) * rstd, o = fmaf(n, w[j][i], bias[j][i]);
        const float dy = in ? cg.v[j].r.at(i) : 0.f;
        float d = dy;
        if (p.gate) {
          const float z1 = cz.v[j].r.at(i), s = sigmoid(z1);
          d = dy * (p.act ? z1 * s : z1);
          dz.r.set(i, dy * o * (p.act ? s * fmaf(z1, 1.f - s, 1.f) : 1.f));
        } else if (p.act) {
          const float s = sigmoid(o);
          d = dy * (s * fmaf(o, 1.f - s, 1.f));
        }
        d = in ? d : 0.f;
        db[j][i] += d;
        dw[j][i] += in ? d * n : 0.f;
        dn[j][i] = d * w[j][i];
        s1 += dn[j][i];
        s2 += in ? dn[j][i] * n : 0.f;
      }
      if (p.gate && have && e < p.W) dz.store((T*)dgate_ + out + e, p.W - e);
    }
    const float m1 = group_sum(s1, p.tpg, red) * (1.f / p.W);
    const float m2 = group_sum(s2, p.tpg, red) * (1.f / p.W);
    if (!have) continue;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (j * p.tpg + at.lane) * 8;
      Cols8<T, VEC> dx;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = (cx.v[j].r.at(i) - mean) * rstd;
        dx.r.set(i, rstd * (dn[j][i] - fmaf(n, m2, m1)));
      }
      if (e < p.W) dx.store((T*)dx_ + out + e, p.W - e);
    }
  }
  if (!part) return;
  // the rb rows' shares of each channel, in order: part [row blocks][2][G W]
  const int per = p.tpg * p.gb, C = p.G * p.W;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) shares[threadIdx.x][i] = at.in ? k ? db[j][i] : dw[j][i] : 0.f;
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * per; i += NORM_THREADS) {
        const int t = i / 8, lane = t % p.tpg, group = blockIdx.y * p.gb + t / p.tpg;
        const int e = (j * p.tpg + lane) * 8 + i % 8;
        if (group >= p.G || e >= p.W) continue;
        float sum = 0.f;
        for (int r = 0; r < p.rb; ++r) sum += shares[r * per + t][i % 8];
        part[((size_t)blockIdx.x * 2 + k) * C + (size_t)group * p.W + e] = sum;
      }
    }
}

// Threads a group: a vector each, up to the workgroup; groups side by side, then rows.
// The rows' blocks bring the forward to eight workgroups a CU (rows in flight hide the two
// sums' latency) and the backward, whose blocks each write a share of dw and db, to four.
void norm_split(Norm& p, bool backward) {
  const int vecs = (p.W + 7) / 8;
  int tpg = 1;
  while (tpg < NORM_THREADS && tpg < vecs) tpg *= 2;
  p.tpg = tpg;
  p.vecs = (vecs + tpg - 1) / tpg;
  int gb = 1;
  while (gb * 2 * tpg <= NORM_THREADS && gb < p.G) gb *= 2;
  p.gb = gb;
  p.rb = NORM_THREADS / (tpg * gb);
  p.group_blocks = (p.G + gb - 1) / gb;
  const long long rows = ((long long)p.batch * p.L + p.rb - 1) / p.rb;
  long long blocks = (backward ? 4LL : 8LL) * device_geom().cus / p.group_blocks;
  if (blocks < 1) blocks = 1;
  p.row_blocks = (int)(rows < blocks ? rows : blocks);
}

#define LZ_NORM_VECS(T, VEC, KERN, ...)                                                        \
  if (p.vecs == 1) hipLaunchKernelGGL((KERN<T, VEC, 1>), grid, block, 0, st, __VA_ARGS__);      \
  else if (p.vecs == 2) hipLaunchKernelGGL((KERN<T, VEC, 2>), grid, block, 0, st, __VA_ARGS__); \
  else hipLaunchKernelGGL((KERN<T, VEC, 4>), grid, block, 0, st, __VA_ARGS__)
#define LZ_NORM_TYPES(KERN, ...)                                                  \
  if (is_bf16 && vec) { LZ_NORM_VECS(bf16, true, KERN, __VA_ARGS__); }            \
  else if (is_bf16) { LZ_NORM_VECS(bf16, false, KERN, __VA_ARGS__); }             \
  else if (vec) { LZ_NORM_VECS(float, true, KERN, __VA_ARGS__); }                 \
  else { LZ_NORM_VECS(float, false, KERN, __VA_ARGS__); }

hipError_t launch_norm_fwd(const Norm& p, bool is_bf16, bool vec, hipStream_t st) {
  const dim3 grid(p.row_blocks, p.group_blocks), block(NORM_THREADS);
  LZ_NORM_TYPES(norm_fwd_kernel, p)
  return hipGetLastError();
}

hipError_t launch_norm_bwd(const Norm& p, const void* dy, void* dx, void* dgate, float* part,
                           float* dw, float* dbias, bool is_bf16, bool vec, hipStream_t st) {
  const dim3 grid(p.row_blocks, p.group_blocks), block(NORM_THREADS);
  LZ_NORM_TYPES(norm_bwd_kernel, p, dy, dx, dgate, part)
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  if (!part) return hipSuccess;
  const int C = p.G * p.W;
  SumJobs jobs = {};
  for (int k = 0; k < 2; ++k)
    if (float* dst = k ? dbias : dw)
      jobs.job[jobs.n++] = SumJob{part + (size_t)k * C, dst, 2LL * C, 0, 0, 1, 1, C, p.row_blocks, 0};
  return launch_sums(jobs, st);
}

}  // namespace lz
