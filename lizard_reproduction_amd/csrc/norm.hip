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
#include <type_traits>

#include "norm.hpp"

namespace lz {

// Sum over the tpg threads of a group (a power of two; past a wave through LDS)
__device__ __forceinline__ float group_sum(float v, int tpg, float* red) {
  v = lanes_sum(v, tpg);
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

// How a thread's vectors meet the group's channels: FULL, the threads' vectors are the
// group; TAIL, the last one is moved back to end with it (its first channels are the vector
// before's), and threads may have none; NARROW, groups of under eight channels, element by
// element.
enum NormFit { FULL, TAIL, NARROW };

// A thread's place: its group, its channels there, and the row it begins with
template <NormFit FIT, int N>
struct NormPlace {
  int slot, lane, group, first[N];
  uint32_t own[N];   // bits: the vector's channels that are this thread's
  bool in;
  __device__ __forceinline__ NormPlace(const Norm& p) {
    lane = threadIdx.x % p.tpg;
    const int i = threadIdx.x / p.tpg;
    slot = i / p.gb;                       // of the rb rows
    group = blockIdx.y * p.gb + i % p.gb;
    in = group < p.G;
    if (!in) group = p.G - 1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = (j * p.tpg + lane) * 8;
      first[j] = FIT == TAIL ? min(e, p.W - 8) : e;
      own[j] = FIT == FULL ? 0xff : FIT == TAIL ? e < p.W ? 0xffu << (e - first[j]) & 0xff : 0
                                                : (1u << p.W) - 1;
    }
  }
  __device__ __forceinline__ bool has(int j, int i) const { return FIT == FULL || own[j] >> i & 1; }
};

// Rows of a tensor of groups, `step` apart, past the last one the last
template <typename T>
struct NormRows {
  const T *p, *last;
  long long step, wrap;   // elements from a row to the next, and more where that passes a sequence
  int left, t, step_t, L;
  __device__ __forceinline__ NormRows(const void* base, long long sb, long long st, long long at,
                                      const Norm& n, int row, int rows_step) {
    const int b = row / n.L;
    L = n.L, t = row - b * L;
    const T* q = (const T*)base + at;
    last = q + (n.batch - 1) * sb + (L - 1) * st;
    p = q + b * sb + t * st;
    step_t = rows_step % L;
    step = rows_step / L * sb + step_t * st;
    wrap = sb - L * st;
    left = n.batch * L - row;   // rows from this one to the end
  }
  __device__ __forceinline__ const T* row() const { return left > 0 ? p : last; }
  __device__ __forceinline__ void next(int rows_step) {
    left -= rows_step;
    p += step;
    t += step_t;
    if (t >= L) t -= L, p += wrap;
  }
};

// f with whether there is a gate and an activation as constants
template <class F>
__device__ __forceinline__ void norm_forms(const Norm& p, F f) {
  using std::false_type;
  using std::true_type;
  if (p.gate) {
    if (p.act) f(true_type(), true_type());
    else f(true_type(), false_type());
  } else {
    if (p.act) f(false_type(), true_type());
    else f(false_type(), false_type());
  }
}

template <typename T, NormFit FIT, int N>
struct NormRow {
  static constexpr bool VEC = FIT != NARROW;
  Cols<T, VEC, 8> v[N];
  __device__ __forceinline__ void load(const T* row, const Norm& p, const int (&first)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j].load(row + first[j], p.W);
  }
};

// the thread's weights and biases
template <NormFit FIT, int N>
__device__ __forceinline__ void norm_params(const Norm& p, const NormPlace<FIT, N>& at,
                                            float (&w)[N][8], float (&bias)[N][8]) {
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float* from = k ? p.bias : p.w;
      Cols<float, FIT != NARROW, 8> v;
      if (from) v.load(from + (size_t)at.group * p.W + at.first[j], p.W);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = from ? v.r.at(i) : k ? 0.f : 1.f;
        if (k) bias[j][i] = x;
        else w[j][i] = x;
      }
    }
}

// mean and 1 / sqrt(var + eps) of a group's row
template <typename T, NormFit FIT, int N>
__device__ __forceinline__ void norm_stats(const NormRow<T, FIT, N>& x, const Norm& p,
                                           const NormPlace<FIT, N>& at, float* red, float& mean,
                                           float& rstd) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += at.has(j, i) ? x.v[j].r.at(i) : 0.f;
  mean = group_sum(sum, p.tpg, red) * p.inv_w;
  sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = at.has(j, i) ? x.v[j].r.at(i) - mean : 0.f;
      sum = fmaf(d, d, sum);
    }
  rstd = __builtin_amdgcn_rsqf(fmaf(group_sum(sum, p.tpg, red), p.inv_w, p.eps));   // within 1 ulp
}

template <typename T, NormFit FIT, int N>
__global__ __launch_bounds__(NORM_THREADS) void norm_fwd_kernel(Norm p) {
  __shared__ float red[4];
  const NormPlace<FIT, N> at(p);
  float w[N][8], bias[N][8];
  norm_params(p, at, w, bias);
  const int rows = p.batch * p.L, step = p.row_blocks * p.rb;
  int row = blockIdx.x * p.rb + at.slot;
  NormRows<T> xr(p.x, p.x_b, p.x_t, at.group * p.x_g, p, row, step);
  NormRows<T> zr(p.gate, p.z_b, p.z_t, at.group * p.z_g, p, row, step);
  NormRow<T, FIT, N> x, z;
  auto load = [&] {
    x.load(xr.row(), p, at.first);
    if (p.gate) z.load(zr.row(), p, at.first);
    xr.next(step);
    if (p.gate) zr.next(step);
  };
  load();
  T* y = (T*)p.y + ((long long)row * p.G + at.group) * p.W;
  const long long y_step = (long long)step * p.G * p.W;
  // every thread makes the same number of rounds: group_sum may hold a barrier
  for (int first = blockIdx.x * p.rb; first < rows; first += step, row += step, y += y_step) {
    const NormRow<T, FIT, N> cx = x, cz = z;
    if (first + step < rows) load();
    float mean, rstd;
    norm_stats(cx, p, at, red, mean, rstd);
    if (!at.in || row >= rows) continue;
    norm_forms(p, [&](auto gate, auto act) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        Cols<T, NormRow<T, FIT, N>::VEC, 8> out;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float o = fmaf((cx.v[j].r.at(i) - mean) * rstd, w[j][i], bias[j][i]);
          const float a = gate.value ? cz.v[j].r.at(i) : o;
          if (act.value) o *= gate.value ? a * sigmoid(a) : sigmoid(a);
          else if (gate.value) o *= a;
          out.r.set(i, o);
        }
        if (at.own[j]) out.store(y + at.first[j], p.W);
      }
    });
  }
}

template <typename T, NormFit FIT, int N>
__global__ __launch_bounds__(NORM_THREADS, N == 1 ? 4 : 1) void norm_bwd_kernel(Norm p, const void* dy_, void* dx_,
                                                                void* dgate_, float* part) {
  __shared__ float red[4];
  __shared__ float shares[NORM_THREADS][9];
  const NormPlace<FIT, N> at(p);
  constexpr bool VEC = NormRow<T, FIT, N>::VEC;
  float w[N][8], bias[N][8], dw[N][8], db[N][8];
  norm_params(p, at, w, bias);
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[j][i] = db[j][i] = 0.f;
  const int rows = p.batch * p.L, step = p.row_blocks * p.rb;
  int row = blockIdx.x * p.rb + at.slot;
  NormRows<T> xr(p.x, p.x_b, p.x_t, at.group * p.x_g, p, row, step);
  NormRows<T> zr(p.gate, p.z_b, p.z_t, at.group * p.z_g, p, row, step);
  long long out = ((long long)row * p.G + at.group) * p.W;   // of dy, dx, dgate
  const long long out_step = (long long)step * p.G * p.W;
  const long long out_last = ((long long)(rows - 1) * p.G + at.group) * p.W;
  NormRow<T, FIT, N> x, z, g;
  auto load = [&](long long o) {
    x.load(xr.row(), p, at.first);
    if (p.gate) z.load(zr.row(), p, at.first);
    g.load((const T*)dy_ + min(o, out_last), p, at.first);
    xr.next(step);
    if (p.gate) zr.next(step);
  };
  load(out);
  for (int first = blockIdx.x * p.rb; first < rows; first += step, row += step, out += out_step) {
    const NormRow<T, FIT, N> cx = x, cz = z, cg = g;
    if (first + step < rows) load(out + out_step);
    float mean, rstd;
    norm_stats(cx, p, at, red, mean, rstd);
    const bool have = at.in && row < rows;
    float s1 = 0.f, s2 = 0.f, dn[N][8];
    norm_forms(p, [&](auto gate, auto act) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        Cols<T, VEC, 8> dz;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = (cx.v[j].r.at(i) - mean) * rstd, o = fmaf(n, w[j][i], bias[j][i]);
          const float dy = cg.v[j].r.at(i);
          float d = dy;
          if (gate.value) {
            const float z1 = cz.v[j].r.at(i), s = sigmoid(z1);
            d = dy * (act.value ? z1 * s : z1);
            dz.r.set(i, dy * o * (act.value ? s * fmaf(z1, 1.f - s, 1.f) : 1.f));
          } else if (act.value) {
            const float s = sigmoid(o);
            d = dy * (s * fmaf(o, 1.f - s, 1.f));
          }
          const float dn1 = d * w[j][i];
          dn[j][i] = dn1;
          if (FIT == FULL) {
            s1 += dn1;
            s2 = fmaf(dn1, n, s2);
          } else {
            s1 += at.has(j, i) ? dn1 : 0.f;
            s2 += at.has(j, i) ? dn1 * n : 0.f;
          }
          d = have ? d : 0.f;   // a row past the last adds nothing
          db[j][i] += d;
          dw[j][i] = fmaf(d, n, dw[j][i]);
        }
        if (gate.value && have && at.own[j]) dz.store((T*)dgate_ + out + at.first[j], p.W);
      }
    });
    const float m1 = group_sum(s1, p.tpg, red) * p.inv_w;
    const float m2 = group_sum(s2, p.tpg, red) * p.inv_w;
    if (!have) continue;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Cols<T, VEC, 8> dx;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = (cx.v[j].r.at(i) - mean) * rstd;
        dx.r.set(i, rstd * (dn[j][i] - fmaf(n, m2, m1)));
      }
      if (at.own[j]) dx.store((T*)dx_ + out + at.first[j], p.W);
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
        int e = (j * p.tpg + lane) * 8;
        if (group >= p.G || e >= p.W) continue;
        if (FIT == TAIL) e = min(e, p.W - 8);   // the overlap: the same sums twice
        e += i % 8;
        if (e >= p.W) continue;
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
  p.inv_w = 1.f / p.W;
  p.group_blocks = (p.G + gb - 1) / gb;
  const long long rows = ((long long)p.batch * p.L + p.rb - 1) / p.rb;
  long long blocks = (backward ? 4LL : 8LL) * device_geom().cus / p.group_blocks;
  if (blocks < 1) blocks = 1;
  p.row_blocks = (int)(rows < blocks ? rows : blocks);
}

#define LZ_NORM_VECS(T, FIT, KERN, ...)                                                        \
  if (p.vecs == 1) hipLaunchKernelGGL((KERN<T, FIT, 1>), grid, block, 0, st, __VA_ARGS__);      \
  else if (p.vecs == 2) hipLaunchKernelGGL((KERN<T, FIT, 2>), grid, block, 0, st, __VA_ARGS__); \
  else hipLaunchKernelGGL((KERN<T, FIT, 4>), grid, block, 0, st, __VA_ARGS__)
#define LZ_NORM_FITS(T, KERN, ...)                                                             \
  if (p.W < 8) hipLaunchKernelGGL((KERN<T, NARROW, 1>), grid, block, 0, st, __VA_ARGS__);       \
  else if (p.W == 8 * p.tpg * (p.vecs > 2 ? 4 : p.vecs)) { LZ_NORM_VECS(T, FULL, KERN, __VA_ARGS__); } \
  else { LZ_NORM_VECS(T, TAIL, KERN, __VA_ARGS__); }
#define LZ_NORM_TYPES(KERN, ...)                  \
  if (is_bf16) { LZ_NORM_FITS(bf16, KERN, __VA_ARGS__) } \
  else { LZ_NORM_FITS(float, KERN, __VA_ARGS__) }

hipError_t launch_norm_fwd(const Norm& p, bool is_bf16, hipStream_t st) {
  const dim3 grid(p.row_blocks, p.group_blocks), block(NORM_THREADS);
  LZ_NORM_TYPES(norm_fwd_kernel, p)
  return hipGetLastError();
}

hipError_t launch_norm_bwd(const Norm& p, const void* dy, void* dx, void* dgate, float* part,
                           float* dw, float* dbias, bool is_bf16, hipStream_t st) {
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
