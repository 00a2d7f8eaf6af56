// Selective state space scan: forward, its pass over segments, and the step of one token.
//
//   delta = softplus(dt + bias), h[n] <- exp(delta A[n]) h[n] + delta x B[n],
//   y = (sum_n C[n] h[n] + D x) silu(z)
//
// for each channel, with B and C shared by a group's channels.  The decay differs for
// every (channel, n), so no run of tokens is a matrix product: per (token, channel, n) it
// takes a product, an exponential, two multiply-adds and the product with B, on the vector
// units, and those bound it, with what the helpers do for each row: B = 4, L = 2048, E = 4096,
// N = 16 in bf16, keeping states for a backward, takes 195 us, the vector units busy 83 % of
// it (the scan's own five instructions are 94 us).  (The products with C on the matrix units,
// as 4 x 4 outer products, were no faster: their operands' layout cost what they saved.)
#include "ssm.hpp"

namespace lz {

// STATE: the segments' own states alone, without C, z and y.
template <typename T, int W, int NP, int NS, int H, bool VEC, bool STATE>
__global__ __launch_bounds__(64 * (W + H)) void ssm_fwd_kernel(Ssm p) {
  constexpr int V = SSM_TILE / (64 * H), COLS = SSM_CH / V;
  // two tiles of each: one worked on by the scan waves, one by the helpers
  __shared__ float sd[2][SSM_TILE], su[2][SSM_TILE], sy[STATE ? 1 : 2 * W][SSM_TILE];
  const int segments = STATE ? p.S - 1 : p.S;
  const SsmPlace at(p, segments);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int E = p.E, N = p.N;
  const long long first = (long long)at.tile0 * SSM_TT;
  auto rows_of = [&](int tile) { return min(SSM_TT, at.len - tile * SSM_TT); };

  // --- rows to delta and u, shares of y to rows (helper) ------------------------------
  const int tid = (int)threadIdx.x - 64 * W;
  const int row = tid / COLS, tc = (tid % COLS) * V, left = at.cols - tc;
  const bool has_z = p.z, soft = p.softplus;
  const int x_t = p.x_t, dt_t = p.dt_t, z_t = p.z_t;
  const T* xb = (const T*)p.x + at.b * p.x_b + first * x_t + at.c0;
  const T* db = (const T*)p.dt + at.b * p.dt_b + first * dt_t + at.c0;
  const T* zb = has_z ? (const T*)p.z + at.b * p.z_b + first * z_t + at.c0 : nullptr;
  T* yb = (T*)p.y + ((long long)at.b * p.L + first) * E + at.c0;
  struct Rows {   // of a tile
    RawRow<T, V, VEC> x, dt, z;
  };
  float bias[V], D[V];
  auto load_params = [&] {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      bias[i] = p.bias && i < left ? p.bias[at.c0 + tc + i] : 0.f;
      D[i] = !STATE && p.D && i < left ? p.D[at.c0 + tc + i] : 0.f;
    }
  };
  auto load_rows = [&](int rows, Rows& r) {
    r.x = load_raw<T, V, VEC>(open_rsrc(xb), row * x_t + tc, row < rows, left);
    r.dt = load_raw<T, V, VEC>(open_rsrc(db), row * dt_t + tc, row < rows, left);
    if (!STATE) r.z = load_raw<T, V, VEC>(open_rsrc(zb), row * z_t + tc, has_z && row < rows, left);
    xb += SSM_TT * (long long)x_t;
    db += SSM_TT * (long long)dt_t;
    if (has_z) zb += SSM_TT * (long long)z_t;
  };
  auto prep = [&](int rows, int buf, const Rows& r) {
    float d[V], u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      d[i] = r.dt.at(i) + bias[i];
      if (soft) d[i] = softplus(d[i]);
      u[i] = d[i] * r.x.at(i);
    }
    if (rows < SSM_TT && row >= rows) {   // past the length: the state stays as it is
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = u[i] = 0.f;
    }
    put_row(sd[buf] + row * SSM_CH + tc, d);
    put_row(su[buf] + row * SSM_CH + tc, u);
  };
  auto finish = [&](int tile, int buf, const RawRow<T, V, VEC>& x, const RawRow<T, V, VEC>& z) {
    const int t0 = tile * SSM_TT, rows = rows_of(tile);
    const rsrc_t ry = open_rsrc(yb);
    float y[V] = {};
#pragma unroll
    for (int j = 0; j < W; ++j) add_row(y, sy[STATE ? 0 : buf * W + j] + row * SSM_CH + tc);
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = fmaf(x.at(i), D[i], y[i]);
    if (has_z) {
      if (p.mixed) {
        RawRow<float, V, VEC> m;
        m.pack(y);
        store_raw<float, V, VEC>(open_rsrc(p.mixed + ((long long)at.b * p.L + t0) * E + at.c0),
                                 row * E + tc, row < rows, left, m);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float g = z.at(i);
        y[i] *= g * sigmoid(g);
      }
    }
    if (rows < SSM_TT && row >= rows) {
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = 0.f;
    }
    RawRow<T, V, VEC> out;
    out.pack(y);
    store_raw<T, V, VEC>(ry, row * E + tc, row < p.L - t0, left, out);
    yb += SSM_TT * (long long)E;
  };

  // --- the walk (scan) ------------------------------------------------------------------
  const int w = wave, c = at.c0 + lane;
  const bool mine = lane < at.cols;
  const int B_t = p.B_t, C_t = p.C_t;
  const T* Bb = (const T*)p.B + at.b * p.B_b + first * B_t + (long long)at.g * p.B_g;
  const T* Cb = (const T*)p.C + at.b * p.C_b + first * C_t + (long long)at.g * p.C_g;
  float* saved = p.saved ? p.saved + ((size_t)at.b * p.tiles + at.tile0) * N * E : nullptr;
  float A2[NP][NS], h[NP][NS], dsum = 0.f;
  SsmVec<T, NS> Bv[NP], Cv[NP];
  auto start = [&] {
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const int n = NS * (w + W * q) + k;
        const bool in = mine && n < N;
        A2[q][k] = in ? p.A[(size_t)c * N + n] * LOG2E : 0.f;
        h[q][k] = in && !STATE && p.state_in ? p.state_in[((size_t)at.b * E + c) * N + n] : 0.f;
      }
    if constexpr (!STATE) {
      // the state before this segment, from the earlier segments' own states
      for (int j = 0; j < at.s; ++j) {
        const size_t rec = (size_t)at.b * (p.S - 1) + j;
        const float d = mine ? p.dsum[rec * E + c] : 0.f;
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int k = 0; k < NS; ++k) {
            const int n = NS * (w + W * q) + k;
            if (mine && n < N)
              h[q][k] = fmaf(__builtin_amdgcn_exp2f(A2[q][k] * d), h[q][k],
                             p.rec[(rec * N + n) * E + c]);
          }
      }
    }
  };
  auto load_bc = [&](int rows) {
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      Bv[q].load(Bb, rows, B_t, N, NS * (w + W * q), lane);
      if (!STATE) Cv[q].load(Cb, rows, C_t, N, NS * (w + W * q), lane);
    }
    Bb += SSM_TT * (long long)B_t;
    Cb += SSM_TT * (long long)C_t;
  };
  float Bf[NP][NS], Cf[NP][NS];
  auto take_bc = [&] {
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        Bf[q][i] = Bv[q].at(i);
        if (!STATE) Cf[q][i] = Cv[q].at(i);
      }
  };
  auto save = [&] {
    if (STATE || !saved) return;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const int n = NS * (w + W * q) + k;
        if (mine && n < N) saved[(size_t)n * E + c] = h[q][k];
      }
    saved += (size_t)N * E;
  };
  auto scan = [&](int buf) {
    constexpr int TOKENS = SsmVec<T, NS>::TOKENS;
    f32x4 dn = get_tokens(sd[buf], 0, lane), un = get_tokens(su[buf], 0, lane);
    static_for<4>([&](auto ki) {
      constexpr int i = decltype(ki)::value;
      const f32x4 dl = dn, ul = un;
      if (i < 3) dn = get_tokens(sd[buf], 4 * i + 4, lane), un = get_tokens(su[buf], 4 * i + 4, lane);
      __builtin_amdgcn_sched_barrier(0);   // the next four tokens' reads go out before these are used
      f32x4 yl;
      if (STATE) dsum += (dl[0] + dl[1]) + (dl[2] + dl[3]);
      static_for<NP>([&](auto kq) {
        constexpr int q = decltype(kq)::value;
        float hs[4][NS];
        static_for<4>([&](auto kt) {
          constexpr int t = decltype(kt)::value, at_t = (4 * i + t) % TOKENS;
          static_for<NS>([&](auto kn) {
            constexpr int n = decltype(kn)::value;
            const float a = __builtin_amdgcn_exp2f(dl[t] * A2[q][n]);
            h[q][n] = fmaf(a, h[q][n],
                           dpp<DPP_BCAST + NS * at_t + n>(Bf[q][4 * i / TOKENS]) * ul[t]);
            hs[t][n] = h[q][n];
          });
        });
        if constexpr (!STATE) ssm_dots<4 * NS * i % 16, (q > 0)>(yl, Cf[q][4 * i / TOKENS], hs);
      });
      if (!STATE) put_tokens(sy[STATE ? 0 : buf * W + w], 4 * i, lane, yl);
    });
  };
  auto end = [&] {
    if (!mine) return;
    const size_t rec = (size_t)at.b * (p.S - 1) + at.s;
    if (STATE && w == 0) p.dsum[rec * E + c] = dsum;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const int n = NS * (w + W * q) + k;
        if (n >= N) continue;
        if (STATE)
          p.rec[(rec * N + n) * E + c] = h[q][k];
        else if (p.state_out && at.s == p.S - 1)
          p.state_out[((size_t)at.b * E + c) * N + n] = h[q][k];
      }
  };

  const int t0 = at.tile0, t1 = at.tile1;   // t0 < t1
  if (wave < W) __builtin_amdgcn_s_setprio(2);   // the scan is the longer of the two
  if (wave >= W) {
    // the rows of two tiles ahead on their way, of this tile and the one before kept to
    // their end; a tile's sums go out after the next rows have come, so that nothing waits
    // for a store
    Rows even, odd, now, last, before;
    load_params();
    load_rows(rows_of(t0), even);
    if (t0 + 1 < t1) load_rows(rows_of(t0 + 1), odd);
    prep(rows_of(t0), 0, even);
    now = even;
    if (t0 + 2 < t1) load_rows(rows_of(t0 + 2), even);
    __syncthreads();
    auto step = [&](int tile, int buf, Rows& next) {
      before = now;
      if (tile + 1 < t1) {
        prep(rows_of(tile + 1), buf ^ 1, next);
        now = next;
        if (tile + 3 < t1) load_rows(rows_of(tile + 3), next);
      }
      if (!STATE && tile > t0) finish(tile - 1, buf ^ 1, last.x, last.z);
      last = before;
      __syncthreads();
    };
    for (int tile = t0; tile < t1; tile += 2) {
      step(tile, 0, odd);
      if (tile + 1 < t1) step(tile + 1, 1, even);
    }
    if (!STATE) finish(t1 - 1, (t1 - 1 - t0) & 1, last.x, last.z);
  } else {
    load_bc(rows_of(t0));
    start();
    __syncthreads();
    for (int tile = t0; tile < t1; ++tile) {
      take_bc();
      if (tile + 1 < t1) load_bc(rows_of(tile + 1));
      save();
      if (rows_of(tile) > 0) scan((tile - t0) & 1);
      __syncthreads();
    }
    end();
  }
}

// One token of R sequences: four lanes to a channel, lane q of them the states 4 q .. 4 q + 3
// of every 16, read and written once as 16 bytes.  The state's bytes bound a large batch (64
// sequences x 4096 channels x 16 states: 9.1 us, 36 MB at 4.0 TB/s), the launch and one round
// of loads a small one (one sequence: 2.9 us).
template <typename T, bool VEC, int R>
__global__ __launch_bounds__(256) void ssm_step_kernel(Ssm p, float* state) {
  const int c = blockIdx.x * 64 + (threadIdx.x >> 2), q = threadIdx.x & 3;
  const bool in = c < p.E;
  const int ci = in ? c : p.E - 1, g = ci / p.Eg;
  const float bias = p.bias ? p.bias[ci] : 0.f, D = p.D ? p.D[ci] : 0.f;
  const float* A = p.A + (size_t)ci * p.N;
  float x[R], d[R], z[R], y[R];
  int b[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    b[r] = min((int)blockIdx.y * R + r, p.batch - 1);   // past the last one, it again
    x[r] = (float)((const T*)p.x)[b[r] * p.x_b + ci];
    d[r] = (float)((const T*)p.dt)[b[r] * p.dt_b + ci];
    z[r] = p.z ? (float)((const T*)p.z)[b[r] * p.z_b + ci] : 0.f;
    y[r] = 0.f;
  }
  for (int n0 = 4 * q; n0 < p.N; n0 += 16) {
    f32x4 h[R], a;
    float Bn[R][4], Cn[R][4];
    if constexpr (VEC) a = *reinterpret_cast<const f32x4*>(A + n0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float* st = state + ((size_t)b[r] * p.E + ci) * p.N;
      const T* B = (const T*)p.B + b[r] * p.B_b + (long long)g * p.B_g;
      const T* C = (const T*)p.C + b[r] * p.C_b + (long long)g * p.C_g;
      if constexpr (VEC) {
        h[r] = *reinterpret_cast<const f32x4*>(st + n0);
        Cols<T, true, 4> b4, c4;
        b4.load(B + n0, 4), c4.load(C + n0, 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) Bn[r][k] = b4.r.at(k), Cn[r][k] = c4.r.at(k);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = min(n0 + k, p.N - 1);
          h[r][k] = st[n];
          a[k] = A[n];
          Bn[r][k] = (float)B[n];
          Cn[r][k] = (float)C[n];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float delta = d[r] + bias;
      if (p.softplus) delta = softplus(delta);
      const float u = delta * x[r];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h[r][k] = fmaf(__builtin_amdgcn_exp2f(delta * (a[k] * LOG2E)), h[r][k], u * Bn[r][k]);
        if (n0 + k < p.N) y[r] = fmaf(Cn[r][k], h[r][k], y[r]);
      }
      float* st = state + ((size_t)b[r] * p.E + ci) * p.N;
      if (in && (R == 1 || (int)blockIdx.y * R + r < p.batch)) {
        if constexpr (VEC) {
          *reinterpret_cast<f32x4*>(st + n0) = h[r];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n0 + k < p.N) st[n0 + k] = h[r][k];
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    y[r] += dpp<DPP_XOR1>(y[r]);
    y[r] += dpp<DPP_XOR2>(y[r]);
    if (q == 0 && in) {
      float o = fmaf(D, x[r], y[r]);
      if (p.z) o *= z[r] * sigmoid(z[r]);
      ((T*)p.y)[(size_t)b[r] * p.E + c] = (T)o;
    }
  }
}

template <typename T, int W, int NP, int NS, int H, bool VEC>
hipError_t fwd_launch(const Ssm& p, hipStream_t st) {
  const int nblk = p.G * p.gblocks;
  const dim3 block(64 * (W + H));
  if (p.S > 1) {
    hipLaunchKernelGGL((ssm_fwd_kernel<T, W, NP, NS, H, VEC, true>),
                       dim3(nblk * (p.S - 1) * p.batch), block, 0, st, p);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((ssm_fwd_kernel<T, W, NP, NS, H, VEC, false>), dim3(nblk * p.S * p.batch),
                     block, 0, st, p);
  return hipGetLastError();
}

// Scan waves W of NS states (and NP passes of them) and helper waves H for N states.  Up to
// eight states a wave takes two, as one wave a SIMD, the channels few or many, is bound by
// its own latency (N = 8, 4096 tokens x 4096 channels: 87 us, with four a wave 124; N = 16,
// eight waves of two against four of four, whose sums and reads of LDS are half as many: 129
// against 125).  Eight scan waves leave room for four helpers where eight would do (N = 32:
// 202 against 214 us; with four scan waves, N = 16, training: 562 with four, 551 with eight).
template <typename T, bool VEC>
hipError_t fwd_waves(const Ssm& p, hipStream_t st) {
  if (p.N <= 4) return fwd_launch<T, 2, 1, 2, 8, VEC>(p, st);
  if (p.N <= 8) return fwd_launch<T, 4, 1, 2, 8, VEC>(p, st);
  if (p.N <= 16) return fwd_launch<T, 4, 1, 4, 8, VEC>(p, st);
  if (p.N <= 32) return fwd_launch<T, 8, 1, 4, 4, VEC>(p, st);
  return fwd_launch<T, 8, 2, 4, 4, VEC>(p, st);
}

// Segments of a sequence.  One where the 64-channel blocks fill the chip, as a pass over
// the segments' own states costs half the walk again (training B = 4, E = 4096, N = 16, 256
// blocks: two segments took 86 us more of 730).  Else as many as bring the forward to two
// workgroups a CU (B = 1, L = 2048, E = 4096: 80, 76, 81 and 83 us at one to four; L =
// 16384, E = 2048: 275, 244, 246, 249), the backward, whose LDS leaves room for one, to one;
// of four tiles at least.
int ssm_segments(int batch, int G, int Eg, int L, bool backward) {
  const int tiles = (L + SSM_TT - 1) / SSM_TT, cus = device_geom().cus;
  const long long groups = (long long)batch * G * ((Eg + SSM_CH - 1) / SSM_CH);
  long long s = groups >= cus ? 1 : backward ? cus / groups : (2 * cus + groups - 1) / groups;
  if (s > tiles / 4) s = tiles / 4;
  if (s > 64) s = 64;
  if (s < 1) s = 1;
  const int seg = (int)((tiles + s - 1) / s);
  return (tiles + seg - 1) / seg;
}

hipError_t launch_ssm_fwd(const Ssm& p, bool is_bf16, bool vec, hipStream_t st) {
  if (is_bf16) return vec ? fwd_waves<bf16, true>(p, st) : fwd_waves<bf16, false>(p, st);
  return vec ? fwd_waves<float, true>(p, st) : fwd_waves<float, false>(p, st);
}

template <typename T, int R>
hipError_t step_launch(const Ssm& p, float* state, hipStream_t st) {
  const dim3 grid((p.E + 63) / 64, (p.batch + R - 1) / R);
  if (p.N % 4 == 0 && ((uintptr_t)state | (uintptr_t)p.A) % 16 == 0)
    hipLaunchKernelGGL((ssm_step_kernel<T, true, R>), grid, dim3(256), 0, st, p, state);
  else
    hipLaunchKernelGGL((ssm_step_kernel<T, false, R>), grid, dim3(256), 0, st, p, state);
  return hipGetLastError();
}

// Two sequences a thread from as many workgroups on as the chip holds at once, eight a CU
// (4096 channels x 16 states: 64 sequences 9.1 us, with one a thread 10.4; 32: 5.9 and 6.2;
// 16: 4.6 and 4.3; one: 3.2 and 2.9)
hipError_t launch_ssm_step(const Ssm& p, float* state, bool is_bf16, hipStream_t st) {
  if ((p.E + 63LL) / 64 * p.batch >= 8LL * device_geom().cus)
    return is_bf16 ? step_launch<bf16, 2>(p, state, st) : step_launch<float, 2>(p, state, st);
  return is_bf16 ? step_launch<bf16, 1>(p, state, st) : step_launch<float, 1>(p, state, st);
}

}  // namespace lz
