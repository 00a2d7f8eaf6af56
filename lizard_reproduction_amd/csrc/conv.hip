// Short causal convolution over the tokens of each channel, channels last:
//
//   pre_t = bias + sum_{j < K} w_j x_{t-K+1+j},   y_t = pre_t or silu(pre_t)
//
// K is at most four, so a value takes a few operations and the bytes of x and y (backward:
// x, dy and dx) bound it.  A thread takes a vector of channels and a run of tokens, with the
// K rows in registers: a row is read once by the run it lies in, and its last K - 1 again,
// from cache, by the run after it.  A workgroup's threads are columns of vectors times runs,
// a row's columns next to each other.  bf16, K = 4, 8192 tokens x 4096 channels: the forward
// takes 28.7 us, 134 MB at 4.7 TB/s, the backward 42.7 us, 201 MB at 4.7 TB/s, where a copy
// runs at 4.9; the last launch, which adds the runs' shares of dw and dbias, 4.6 us.
//
// Backward: g_t = dy_t act'(pre_t), dx_t = sum_j w_j g_{t+K-1-j} (the run goes K - 1 tokens
// on), dw_j = sum_t g_t x_{t-K+1+j}, dbias = sum_t g_t: the workgroup's runs meet in LDS and
// its shares go to a second launch, which adds them in order.
#include <type_traits>

#include "conv.hpp"

namespace lz {

// Where a thread works: its columns, and its run of tokens of a sequence
template <int V, bool VEC>
struct ConvPlace {
  int col, run, b, t0, left;
  bool in;
  __device__ __forceinline__ ConvPlace(const Conv& p) {
    col = (blockIdx.y * p.cols + threadIdx.x % p.cols) * V;
    run = blockIdx.x * (CONV_THREADS / p.cols) + threadIdx.x / p.cols;
    in = col < p.C && run < p.batch * p.seq_runs;
    if (!in) col = 0, run = 0;
    if (VEC && col + V > p.C) col = p.C - V;   // the last vector overlaps the one before
    b = run / p.seq_runs;
    t0 = (run - b * p.seq_runs) * p.run;
    left = p.C - col;
  }
};

template <int K, int V, bool VEC>
__device__ __forceinline__ void load_taps(const Conv& p, int col, int left, float (&w)[K][V],
                                          float (&bias)[V]) {
  if constexpr (VEC) {   // the channels' taps lie next to each other
    Cols<float, true, V * K> t;
    t.load(p.w + (size_t)col * K, V * K);
    Cols<float, true, V> b;
    if (p.bias) b.load(p.bias + col, V);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][i] = t.r.at(i * K + j);
      bias[i] = p.bias ? b.r.at(i) : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = col + (i < left ? i : 0);
#pragma unroll
      for (int j = 0; j < K; ++j) w[j][i] = p.w[(size_t)c * K + j];
      bias[i] = p.bias ? p.bias[c] : 0.f;
    }
  }
}

// Row t of sequence b, from the kept state where t < 0 (zeros without one)
template <typename T, bool VEC, int K, int V>
__device__ __forceinline__ void row_before(const Conv& p, const T* xb, int b, int t, int col,
                                           int left, float (&v)[V]) {
  Cols<T, VEC, V> c;
  const T* state = (const T*)p.state_in;
  const bool have = t >= 0 || state;
  const T* from = t >= 0 || !state ? xb + (long long)max(t, 0) * p.x_t
                                   : state + ((long long)b * (K - 1) + (t + K - 1)) * p.C + col;
  c.load(from, left);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = have ? c.r.at(i) : 0.f;
}

constexpr int CONV_AHEAD = 4;   // rows on their way while as many are worked on

template <typename T, bool VEC, int K>
__global__ __launch_bounds__(CONV_THREADS) void conv_fwd_kernel(Conv p) {
  constexpr int V = CONV_FWD_V;
  const ConvPlace<V, VEC> at(p);
  if (!at.in) return;
  const int len = p.lengths ? max(0, min(p.L, p.lengths[at.b])) : p.L;
  const T* xb = (const T*)p.x + at.b * p.x_b + at.col;
  T* yb = (T*)p.y + (long long)at.b * p.L * p.C + at.col;
  float w[K][V], bias[V], win[K][V];   // win[j]: row t - K + 1 + j
  load_taps<K, V, VEC>(p, at.col, at.left, w, bias);
#pragma unroll
  for (int j = 1; j < K; ++j)
    row_before<T, VEC, K, V>(p, xb, at.b, at.t0 + j - K, at.col, at.left, win[j]);
  const int t1 = min(at.t0 + p.run, p.L);
  Cols<T, VEC, V> next[CONV_AHEAD];   // a batch of rows on its way while one is worked on
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < CONV_AHEAD; ++i)
      next[i].load(xb + (long long)min(t + i, p.L - 1) * p.x_t, at.left);
  };
  load(at.t0);
  for (int t = at.t0; t < t1; t += CONV_AHEAD) {
    Cols<T, VEC, V> x[CONV_AHEAD];
#pragma unroll
    for (int i = 0; i < CONV_AHEAD; ++i) x[i] = next[i];
    if (t + CONV_AHEAD < t1) load(t + CONV_AHEAD);
#pragma unroll
    for (int i = 0; i < CONV_AHEAD; ++i) {
      Cols<T, VEC, V> out;
      float ys[V];
#pragma unroll
      for (int c = 0; c < V; ++c) {
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) win[j][c] = win[j + 1][c];
        win[K - 1][c] = x[i].r.at(c);
        float y = bias[c];
#pragma unroll
        for (int j = 0; j < K; ++j) y = fmaf(w[j][c], win[j][c], y);
        if (p.act) y *= sigmoid(y);
        ys[c] = t + i < len ? y : 0.f;
      }
      out.r.pack(ys);
      if (t + i < t1) out.store(yb + (long long)(t + i) * p.C, at.left);
    }
  }
  // the last K - 1 rows of the sequence, by the run that begins it
  if (K > 1 && p.state_out && at.t0 == 0) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      float v[V];
      row_before<T, VEC, K, V>(p, xb, at.b, len - (K - 1) + j, at.col, at.left, v);
      Cols<T, VEC, V> out;
      out.r.pack(v);
      out.store((T*)p.state_out + ((long long)at.b * (K - 1) + j) * p.C + at.col, at.left);
    }
  }
}

// One token of each sequence: a thread a channel, its kept rows moved up in place.  One
// round of loads and the launch bound it (2.6 us at one sequence of 2048 channels).
template <typename T, int K>
__global__ __launch_bounds__(256) void conv_step_kernel(Conv p) {
  const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (c >= p.C) return;
  T* state = (T*)p.state_out + (long long)b * (K - 1) * p.C + c;
  T row[K];
#pragma unroll
  for (int j = 0; j < K - 1; ++j) row[j] = state[(long long)j * p.C];
  row[K - 1] = ((const T*)p.x)[b * p.x_b + c];
  float y = p.bias ? p.bias[c] : 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j) y = fmaf(p.w[(size_t)c * K + j], (float)row[j], y);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) state[(long long)j * p.C] = row[j + 1];
  if (p.act) y *= sigmoid(y);
  ((T*)p.y)[(long long)b * p.C + c] = (T)y;
}

template <typename T, bool VEC, int K>
__global__ __launch_bounds__(CONV_THREADS) void conv_bwd_kernel(Conv p, const void* dy_, void* dx_,
                                                                float* part) {
  constexpr int V = CONV_BWD_V;
  __shared__ float red[CONV_THREADS][V + 1];
  const ConvPlace<V, VEC> at(p);
  const T* xb = (const T*)p.x + at.b * p.x_b + at.col;
  const T* dyb = (const T*)dy_ + (long long)at.b * p.L * p.C + at.col;
  T* dxb = (T*)dx_ + (long long)at.b * p.L * p.C + at.col;
  float w[K][V], bias[V], win[K][V], g[K][V];   // g[j]: the gradient at token t - K + 1 + j
  float dw[K][V], dbias[V];
  load_taps<K, V, VEC>(p, at.col, at.left, w, bias);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    dbias[c] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) dw[j][c] = g[j][c] = 0.f;
  }
#pragma unroll
  for (int j = 1; j < K; ++j)
    row_before<T, VEC, K, V>(p, xb, at.b, at.t0 + j - K, at.col, at.left, win[j]);
  // Token t's row: its gradient g, this run's share of dw and dbias (OWN), and dx of token
  // t - K + 1, the last whose taps are complete.  Past the sequence g is zero.
  const int t1 = at.in ? min(at.t0 + p.run, p.L) : at.t0;
  auto row = [&](int t, const Cols<T, VEC, V>& x, const Cols<T, VEC, V>& dy, auto own) {
    Cols<T, VEC, V> out;
    float dxs[V];
    const bool there = t < p.L;
#pragma unroll
    for (int c = 0; c < V; ++c) {
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) win[j][c] = win[j + 1][c], g[j][c] = g[j + 1][c];
      win[K - 1][c] = x.r.at(c);
      float d = dy.r.at(c);
      if (p.act) {
        float pre = bias[c];
#pragma unroll
        for (int j = 0; j < K; ++j) pre = fmaf(w[j][c], win[j][c], pre);
        const float s = sigmoid(pre);
        d *= s * fmaf(pre, 1.f - s, 1.f);
      }
      d = there ? d : 0.f;
      g[K - 1][c] = d;
      if (decltype(own)::value) dbias[c] += d;
      float dx = 0.f;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (decltype(own)::value) dw[j][c] = fmaf(d, win[j][c], dw[j][c]);
        dx = fmaf(w[j][c], g[K - 1 - j][c], dx);   // g at token t - j: tap K - 1 - j
      }
      dxs[c] = dx;
    }
    out.r.pack(dxs);
    const int to = t - (K - 1);
    if (to >= at.t0 && to < t1) out.store(dxb + (long long)to * p.C, at.left);
  };
  auto load = [&](int t, Cols<T, VEC, V>& x, Cols<T, VEC, V>& dy) {
    const long long r = min(t, p.L - 1);
    x.load(xb + r * p.x_t, at.left);
    dy.load(dyb + r * p.C, at.left);
  };
  // A run is whole batches of rows, but the last one, whose rows past it are past the
  // sequence; a batch is on its way while one is worked on
  Cols<T, VEC, V> nx[CONV_AHEAD], ny[CONV_AHEAD];
  auto load_batch = [&](int t) {
#pragma unroll
    for (int i = 0; i < CONV_AHEAD; ++i) load(t + i, nx[i], ny[i]);
  };
  static_assert(CONV_AHEAD >= CONV_MAX_TAPS - 1, "a batch holds the rows after a run");
  int t = at.t0;
  load_batch(t);
  for (; t < t1; t += CONV_AHEAD) {
    Cols<T, VEC, V> x[CONV_AHEAD], dy[CONV_AHEAD];
#pragma unroll
    for (int i = 0; i < CONV_AHEAD; ++i) x[i] = nx[i], dy[i] = ny[i];
    load_batch(t + CONV_AHEAD);
#pragma unroll
    for (int i = 0; i < CONV_AHEAD; ++i) row(t + i, x[i], dy[i], std::true_type());
  }
  if (at.in) {   // the tokens after the run that its last rows reach
#pragma unroll
    for (int i = 0; i < K - 1; ++i) row(t + i, nx[i], ny[i], std::false_type());
  }
  // the workgroup's runs, one sum at a time: [K + 1][C] floats a row of workgroups
  const int runs = CONV_THREADS / p.cols;
#pragma unroll
  for (int j = 0; j <= K; ++j) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < V; ++c) red[threadIdx.x][c] = j < K ? dw[j < K ? j : 0][c] : dbias[c];
    __syncthreads();
    for (int i = threadIdx.x; i < V * p.cols; i += CONV_THREADS) {
      const int t = i / V;   // the threads of a column of vectors
      int ch = (blockIdx.y * p.cols + t) * V;
      if (ch >= p.C) continue;
      if (VEC && ch + V > p.C) ch = p.C - V;
      ch += i % V;
      if (ch >= p.C) continue;
      float sum = 0.f;
      for (int r = 0; r < runs; ++r) sum += red[r * p.cols + t][i % V];
      part[((size_t)blockIdx.x * (K + 1) + j) * p.C + ch] = sum;
    }
  }
}

// Runs long enough that their K - 1 rows before them cost little, short enough that the
// threads fill the chip: two workgroups a CU in the forward (8192 tokens x 4096 channels: 28.9
// us, with 1.5, 3 and 4 a CU 32.7, 31.0 and 33.1), four in the backward (42.7 us, with 2, 3
// and 8 45.4, 43.9 and 47.3).  Runs of at most 32, 64 and 128 tokens made 1 % of a difference.
void conv_split(Conv& p, bool backward) {
  const int V = backward ? CONV_BWD_V : CONV_FWD_V, vecs = (p.C + V - 1) / V;
  int cols = 1;
  while (cols < 64 && cols < vecs) cols *= 2;
  // fewer where the last block of columns would be mostly empty (2050 channels: 15 us, with
  // 64 columns all the same 23)
  while (cols > 16 && (vecs + cols - 1) / cols * cols * 8 > vecs * 9) cols /= 2;
  p.cols = cols;
  p.col_blocks = (vecs + cols - 1) / cols;
  const long long rows = (long long)p.batch * p.L;
  const long long threads = (backward ? 1024LL : 512LL) * device_geom().cus;
  long long run = rows * vecs / threads;
  run = run < 8 ? 8 : run > 64 ? 64 : run;
  run = (run + CONV_AHEAD - 1) / CONV_AHEAD * CONV_AHEAD;
  p.run = (int)run;
  p.seq_runs = (int)((p.L + run - 1) / run);
  const long long all = (long long)p.batch * p.seq_runs, per = CONV_THREADS / cols;
  p.run_blocks = (int)((all + per - 1) / per);
}

template <typename T, bool VEC>
hipError_t conv_taps(const Conv& p, int K, const void* dy, void* dx, float* part, hipStream_t st) {
  const dim3 grid(p.run_blocks, p.col_blocks), block(CONV_THREADS);
#define LZ_TAPS(k)                                                                        \
  if (K == k) {                                                                           \
    if (dy) hipLaunchKernelGGL((conv_bwd_kernel<T, VEC, k>), grid, block, 0, st, p, dy, dx, part); \
    else hipLaunchKernelGGL((conv_fwd_kernel<T, VEC, k>), grid, block, 0, st, p);         \
  }
  LZ_TAPS(1) LZ_TAPS(2) LZ_TAPS(3) LZ_TAPS(4)
#undef LZ_TAPS
  return hipGetLastError();
}

hipError_t launch_conv(const Conv& p, int K, const void* dy, void* dx, float* part, bool is_bf16,
                       bool vec, hipStream_t st) {
  if (is_bf16)
    return vec ? conv_taps<bf16, true>(p, K, dy, dx, part, st)
               : conv_taps<bf16, false>(p, K, dy, dx, part, st);
  return vec ? conv_taps<float, true>(p, K, dy, dx, part, st)
             : conv_taps<float, false>(p, K, dy, dx, part, st);
}

hipError_t launch_conv_sums(const Conv& p, int K, const float* part, float* dw, float* dbias,
                            hipStream_t st) {
  SumJobs jobs = {};
  // part [parts][K + 1][C] -> dw [C, K], dbias [C]
  jobs.job[jobs.n++] = SumJob{part, dw, (long long)(K + 1) * p.C, p.C, 1, K, K, p.C, p.run_blocks, 0};
  if (dbias)
    jobs.job[jobs.n++] = SumJob{part + (size_t)K * p.C, dbias, (long long)(K + 1) * p.C, 0, 0, 1, 1,
                                p.C, p.run_blocks, 0};
  return launch_sums(jobs, st);
}

template <typename T>
hipError_t step_taps(const Conv& p, int K, hipStream_t st) {
  const dim3 grid((p.C + 255) / 256, p.batch);
#define LZ_TAPS(k) \
  if (K == k) hipLaunchKernelGGL((conv_step_kernel<T, k>), grid, dim3(256), 0, st, p);
  LZ_TAPS(1) LZ_TAPS(2) LZ_TAPS(3) LZ_TAPS(4)
#undef LZ_TAPS
  return hipGetLastError();
}

hipError_t launch_conv_step(const Conv& p, int K, bool is_bf16, hipStream_t st) {
  return is_bf16 ? step_taps<bf16>(p, K, st) : step_taps<float>(p, K, st);
}

}  // namespace lz
