// Normalisation of groups of channels of each token, with an affine map and an activation:
//
//   n = (x - mean) / sqrt(var + eps) over the group's W channels,  o = n w + b,
//   y = o, silu(o), o gate or o silu(gate)
//
// A group is read once into the registers of as many threads as it has vectors of eight
// channels, its mean and then its squared distances from it summed across them in fp32, so
// the rows' bytes bound it (bf16, 8192 tokens of 32 groups of 128, with a gate: the forward
// takes 43 us, 201 MB at 4.7 TB/s, the backward 65 us, 335 MB at 5.1 TB/s, where a copy runs at
// 4.9).  A thread keeps its channels, with w and b (backward: the sums of dw and db) in
// registers, and goes through rows; the next row's loads are issued before this row is
// worked on.  Groups may lie apart by any stride (the heads of an attention
// output); y is rows.
//
// Backward, from x again: do = dy act', dn = do w, dx = (dn - mean(dn) - n mean(dn n)) rstd,
// dgate = dy o act'(gate), dw = sum do n, db = sum do.  A workgroup's shares of dw and db go
// to a second launch, which adds them in order.
#include <type_traits>

#include "norm.hpp"

namespace lz {

// Sums over the tpg threads of a group (a power of two; past a wave through LDS)
template <int S>
__device__ __forceinline__ void group_sums(float (&v)[S], int tpg, float (&red)[S][4]) {
  lanes_sum(v, tpg);
  if (tpg > 64) {   // uniform
    const int wave = threadIdx.x >> 6, per = tpg >> 6;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < S; ++k)
      if ((threadIdx.x & 63) == 0) red[k][wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < S; ++k) {
      v[k] = 0.f;
      for (int i = 0; i < per; ++i) v[k] += red[k][wave / per * per + i];
    }
  }
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

// A walk over rows `step` apart in x and the gate, past the last one the last
template <typename T, bool GATE>
struct NormWalk {
  static constexpr int M = GATE ? 2 : 1;
  const T *p[M], *last[M];
  long long step[M], wrap[M];   // elements to the next row, and more where that passes a sequence
  int left, t, step_t, L;
  __device__ __forceinline__ NormWalk(const Norm& n, int group, int row, int rows_step) {
    const int b = row / n.L;
    L = n.L, t = row - b * L;
    step_t = rows_step % L;
    left = n.batch * L - row;   // rows from this one to the end
#pragma unroll
    for (int k = 0; k < M; ++k) {
      const long long sb = k ? n.z_b : n.x_b, st = k ? n.z_t : n.x_t, sg = k ? n.z_g : n.x_g;
      const T* q = (const T*)(k ? n.gate : n.x) + group * sg;
      last[k] = q + (n.batch - 1) * sb + (L - 1) * st;
      p[k] = q + b * sb + t * st;
      step[k] = rows_step / L * sb + step_t * st;
      wrap[k] = sb - L * st;
    }
  }
  __device__ __forceinline__ const T* row(int k) const { return left > 0 ? p[k] : last[k]; }
  __device__ __forceinline__ void next(int rows_step) {
    left -= rows_step;
    t += step_t;
    const bool over = t >= L;
    if (over) t -= L;
#pragma unroll
    for (int k = 0; k < M; ++k) p[k] += over ? step[k] + wrap[k] : step[k];
  }
};

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
                                           const NormPlace<FIT, N>& at, float (&red)[1][4], float& mean,
                                           float& rstd) {
  float sum[1] = {0.f};
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[0] += at.has(j, i) ? x.v[j].r.at(i) : 0.f;
  group_sums(sum, p.tpg, red);
  mean = sum[0] * p.inv_w;
  sum[0] = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = at.has(j, i) ? x.v[j].r.at(i) - mean : 0.f;
      sum[0] = fmaf(d, d, sum[0]);
    }
  group_sums(sum, p.tpg, red);
  rstd = __builtin_amdgcn_rsqf(fmaf(sum[0], p.inv_w, p.eps));   // within 1 ulp
}

// The gate and the activation are template arguments: as branches in the loops over elements
// they took the backward's walk 84 us where it now takes 65.
template <typename T, NormFit FIT, int N, bool GATE, bool ACT>
__global__ __launch_bounds__(NORM_THREADS) void norm_fwd_kernel(Norm p) {
  __shared__ float red[1][4];
  const NormPlace<FIT, N> at(p);
  float w[N][8], bias[N][8];
  norm_params(p, at, w, bias);
  const int rows = p.batch * p.L, step = p.row_blocks * p.rb;
  int row = blockIdx.x * p.rb + at.slot;
  NormWalk<T, GATE> walk(p, at.group, row, step);
  struct Rows {
    NormRow<T, FIT, N> x, z;
  };
  auto load = [&](Rows& r) {
    r.x.load(walk.row(0), p, at.first);
    if constexpr (GATE) r.z.load(walk.row(1), p, at.first);
    walk.next(step);
  };
  T* y = (T*)p.y + ((long long)row * p.G + at.group) * p.W;
  const long long y_step = (long long)step * p.G * p.W;
  auto work = [&](const Rows& r) {
    float mean, rstd;
    norm_stats(r.x, p, at, red, mean, rstd);
    if (!at.in || row >= rows) return;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Cols<T, NormRow<T, FIT, N>::VEC, 8> out;
      float os[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float o = fmaf((r.x.v[j].r.at(i) - mean) * rstd, w[j][i], bias[j][i]);
        const float a = GATE ? r.z.v[j].r.at(i) : o;
        if (ACT) o *= GATE ? a * sigmoid(a) : sigmoid(a);
        else if (GATE) o *= a;
        os[i] = o;
      }
      out.r.pack(os);
      if (at.own[j]) out.store(y + at.first[j], p.W);
    }
  };
  // Two rows by turns, one on its way while the other is worked on; every thread makes the
  // same number of rounds, as a group's sums may hold a barrier
  Rows even, odd;
  load(even);
  int first = blockIdx.x * p.rb;
  auto round = [&](const Rows& now, Rows& next) {
    const bool more = first + step < rows;
    if (more) load(next);
    work(now);
    first += step, row += step, y += y_step;
    return more;
  };
  while (round(even, odd) && round(odd, even)) {
  }
}

template <typename T, NormFit FIT, int N, bool GATE, bool ACT>
__global__ __launch_bounds__(NORM_THREADS, N == 1 ? 4 : 1) void norm_bwd_kernel(
    Norm p, const void* dy_, void* dx_, void* dgate_, float* part) {
  __shared__ float red[1][4], red2[2][4];
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
  NormWalk<T, GATE> walk(p, at.group, row, step);
  long long out = ((long long)row * p.G + at.group) * p.W;   // of dy, dx, dgate
  const long long out_step = (long long)step * p.G * p.W;
  const long long out_last = ((long long)(rows - 1) * p.G + at.group) * p.W;
  struct Rows {
    NormRow<T, FIT, N> x, z, g;
  };
  auto load = [&](Rows& r, long long o) {
    r.x.load(walk.row(0), p, at.first);
    if constexpr (GATE) r.z.load(walk.row(1), p, at.first);
    r.g.load((const T*)dy_ + min(o, out_last), p, at.first);
    walk.next(step);
  };
  auto work = [&](const Rows& r) {
    float mean, rstd;
    norm_stats(r.x, p, at, red, mean, rstd);
    const bool have = at.in && row < rows;
    float s[2] = {0.f, 0.f}, dn[N][8];   // of dn and of dn n
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Cols<T, VEC, 8> dz;
      float dzs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = (r.x.v[j].r.at(i) - mean) * rstd, o = fmaf(n, w[j][i], bias[j][i]);
        const float dy = r.g.v[j].r.at(i);
        float d = dy;
        if (GATE) {
          const float z1 = r.z.v[j].r.at(i), a = sigmoid(z1);
          d = dy * (ACT ? z1 * a : z1);
          dzs[i] = dy * o * (ACT ? a * fmaf(z1, 1.f - a, 1.f) : 1.f);
        } else if (ACT) {
          const float a = sigmoid(o);
          d = dy * (a * fmaf(o, 1.f - a, 1.f));
        }
        const float dn1 = d * w[j][i];
        dn[j][i] = dn1;
        if (FIT == FULL) {
          s[0] += dn1;
          s[1] = fmaf(dn1, n, s[1]);
        } else {
          s[0] += at.has(j, i) ? dn1 : 0.f;
          s[1] += at.has(j, i) ? dn1 * n : 0.f;
        }
        d = have ? d : 0.f;   // a row past the last adds nothing
        db[j][i] += d;
        dw[j][i] = fmaf(d, n, dw[j][i]);
      }
      if (GATE) dz.r.pack(dzs);
      if (GATE && have && at.own[j]) dz.store((T*)dgate_ + out + at.first[j], p.W);
    }
    group_sums(s, p.tpg, red2);
    if (!have) return;
    const float m1 = s[0] * p.inv_w, m2 = s[1] * p.inv_w;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Cols<T, VEC, 8> dx;
      float dxs[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = (r.x.v[j].r.at(i) - mean) * rstd;
        dxs[i] = rstd * (dn[j][i] - fmaf(n, m2, m1));
      }
      dx.r.pack(dxs);
      if (at.own[j]) dx.store((T*)dx_ + out + at.first[j], p.W);
    }
  };
  Rows even, odd;
  load(even, out);
  int first = blockIdx.x * p.rb;
  auto round = [&](const Rows& now, Rows& next) {   // as in the forward
    const bool more = first + step < rows;
    if (more) load(next, out + out_step);
    work(now);
    first += step, row += step, out += out_step;
    return more;
  };
  while (round(even, odd) && round(odd, even)) {
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
// The rows' blocks bring the forward to eight workgroups a CU (3063 tokens of 32 groups of
// 64: 9.8 us; with 4 and 16 a CU 10.3 and 10.6) and the backward, whose blocks each write a
// share of dw and db, to four (8192 tokens of 32 groups of 128, with the shares' sums: 68 us
// with 2 and 4, 84 with 8).
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

template <typename T, NormFit FIT_, int N_>
struct NormForm {
  using type = T;
  static constexpr NormFit FIT = FIT_;
  static constexpr int N = N_;
};
// Calls f with the template arguments that p and the type ask for
template <typename T, NormFit FIT, int N, class F>
void norm_forms(const Norm& p, F f) {
  using A = NormForm<T, FIT, N>;
  if (p.gate) {
    if (p.act) f(A(), std::true_type(), std::true_type());
    else f(A(), std::true_type(), std::false_type());
  } else {
    if (p.act) f(A(), std::false_type(), std::true_type());
    else f(A(), std::false_type(), std::false_type());
  }
}
template <typename T, NormFit FIT, class F>
void norm_vecs(const Norm& p, F f) {
  if (p.vecs == 1) norm_forms<T, FIT, 1>(p, f);
  else if (p.vecs == 2) norm_forms<T, FIT, 2>(p, f);
  else norm_forms<T, FIT, 4>(p, f);
}
template <typename T, class F>
void norm_fits(const Norm& p, F f) {
  if (p.W < 8) norm_forms<T, NARROW, 1>(p, f);
  else if (p.W == 8 * p.tpg * (p.vecs > 2 ? 4 : p.vecs)) norm_vecs<T, FULL>(p, f);
  else norm_vecs<T, TAIL>(p, f);
}
template <class F>
void norm_types(const Norm& p, bool is_bf16, F f) {
  if (is_bf16) norm_fits<bf16>(p, f);
  else norm_fits<float>(p, f);
}

hipError_t launch_norm_fwd(const Norm& p, bool is_bf16, hipStream_t st) {
  const dim3 grid(p.row_blocks, p.group_blocks), block(NORM_THREADS);
  norm_types(p, is_bf16, [&](auto form, auto gate, auto act) {
    using A = decltype(form);
    hipLaunchKernelGGL((norm_fwd_kernel<typename A::type, A::FIT, A::N, gate.value, act.value>), grid,
                       block, 0, st, p);
  });
  return hipGetLastError();
}

hipError_t launch_norm_bwd(const Norm& p, const void* dy, void* dx, void* dgate, float* part,
                           float* dw, float* dbias, bool is_bf16, hipStream_t st) {
  const dim3 grid(p.row_blocks, p.group_blocks), block(NORM_THREADS);
  norm_types(p, is_bf16, [&](auto form, auto gate, auto act) {
    using A = decltype(form);
    hipLaunchKernelGGL((norm_bwd_kernel<typename A::type, A::FIT, A::N, gate.value, act.value>), grid,
                       block, 0, st, p, dy, dx, dgate, part);
  });
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
