// Selective state space scan: forward, its pass over segments, and the step of one token.
//
//   delta = softplus(dt + bias), h[n] <- exp(delta A[n]) h[n] + delta x B[n],
//   y = (sum_n C[n] h[n] + D x) silu(z)
//
// for each channel, with B and C shared by a group's channels.  The decay differs for
// every (channel, n), so no run of tokens is a matrix product: per (token, channel, n) it
// takes a product, an exponential, two multiply-adds and the product with B, on the vector
// units, and those bound it.
#include "ssm.hpp"

namespace lz {

template <typename T, int W, int NP, bool VEC, bool STATE>
__global__ __launch_bounds__(64 * W) void ssm_fwd_kernel(Ssm p) {
  using Split = SsmSplit<W>;
  constexpr int V = Split::V, R = Split::R;
  __shared__ float sd[SSM_TILE], su[SSM_TILE], sy[STATE ? 1 : W * SSM_TILE];
  const int segments = STATE ? p.S - 1 : p.S;
  const SsmPlace at(p, segments);
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = at.c0 + lane;
  const bool mine = lane < at.cols;

  float A2[NP][4], h[NP][4];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = 4 * (w + W * q) + k;
      const bool in = mine && n < p.N;
      A2[q][k] = in ? p.A[(size_t)c * p.N + n] * LOG2E : 0.f;
      h[q][k] = in && !STATE && p.state_in ? p.state_in[((size_t)at.b * p.E + c) * p.N + n] : 0.f;
    }
  if constexpr (!STATE) {
    // the state before this segment, from the earlier segments' own states
    for (int j = 0; j < at.s; ++j) {
      const size_t rec = (size_t)at.b * (p.S - 1) + j;
      const float d = mine ? p.dsum[rec * p.E + c] : 0.f;
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = 4 * (w + W * q) + k;
          if (mine && n < p.N)
            h[q][k] = fmaf(__builtin_amdgcn_exp2f(A2[q][k] * d), h[q][k],
                           p.rec[(rec * p.N + n) * p.E + c]);
        }
    }
  }

  // this thread's share of a tile's rows
  const int tr = tid / Split::COLS, tc = (tid % Split::COLS) * V, left = at.cols - tc;
  float bias[V], D[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = p.bias && i < left ? p.bias[at.c0 + tc + i] : 0.f;
    D[i] = !STATE && p.D && i < left ? p.D[at.c0 + tc + i] : 0.f;
  }
  // where the next tile's rows begin, and from one tile to the next
  const long long first = (long long)at.tile0 * SSM_TT;
  const T* xb = (const T*)p.x + at.b * p.x_b + first * p.x_t + at.c0;
  const T* db = (const T*)p.dt + at.b * p.dt_b + first * p.dt_t + at.c0;
  const T* zb = p.z ? (const T*)p.z + at.b * p.z_b + first * p.z_t + at.c0 : nullptr;
  const T* Bb = (const T*)p.B + at.b * p.B_b + first * p.B_t + (long long)at.g * p.B_g;
  const T* Cb = (const T*)p.C + at.b * p.C_b + first * p.C_t + (long long)at.g * p.C_g;
  T* yb = (T*)p.y + ((long long)at.b * p.L + first) * p.E + at.c0;
  float* saved = p.saved ? p.saved + ((size_t)at.b * p.tiles + at.tile0) * p.N * p.E : nullptr;
  const size_t saved_step = (size_t)p.N * p.E;
  const int x_t = p.x_t, dt_t = p.dt_t, z_t = p.z_t, B_t = p.B_t, C_t = p.C_t, E = p.E, N = p.N;
  const bool has_z = p.z, soft = p.softplus;

  RawRow<T, V, VEC> xr[R], dr[R], zr[R];
  SsmVec<T> Bv[NP], Cv[NP];
  auto load = [&](int rows) {
    const rsrc_t rx = open_rsrc(xb), rd = open_rsrc(db), rz = open_rsrc(zb);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = tr + r * Split::ROWS;
      xr[r] = load_raw<T, V, VEC>(rx, row * x_t + tc, row < rows, left);
      dr[r] = load_raw<T, V, VEC>(rd, row * dt_t + tc, row < rows, left);
      if (!STATE) zr[r] = load_raw<T, V, VEC>(rz, row * z_t + tc, has_z && row < rows, left);
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      Bv[q].load(Bb, rows, B_t, N, 4 * (w + W * q), lane);
      if (!STATE) Cv[q].load(Cb, rows, C_t, N, 4 * (w + W * q), lane);
    }
    xb += SSM_TT * (long long)x_t;
    db += SSM_TT * (long long)dt_t;
    if (has_z) zb += SSM_TT * (long long)z_t;
    Bb += SSM_TT * (long long)B_t;
    Cb += SSM_TT * (long long)C_t;
  };

  float dsum = 0.f;
  if (at.tile0 < at.tile1) load(min(SSM_TT, at.len - at.tile0 * SSM_TT));
  for (int tile = at.tile0; tile < at.tile1; ++tile) {
    const int t0 = tile * SSM_TT;
    const int rows = min(SSM_TT, at.len - t0);
    float xv[R][V], gate[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = tr + r * Split::ROWS;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = xr[r].at(i);
        float d = dr[r].at(i) + bias[i];
        if (soft) d = softplus(d);
        if (row >= rows) d = 0.f;   // past the length: the state stays as it is
        sd[(tc + i) * SSM_PITCH + row] = d;
        su[(tc + i) * SSM_PITCH + row] = d * x;
        xv[r][i] = x * D[i];
        if (!STATE) {
          const float z = zr[r].at(i);
          gate[r][i] = has_z ? z * sigmoid(z) : 1.f;
        }
      }
    }
    float Bf[NP][4], Cf[NP][4];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Bf[q][i] = Bv[q].at(i);
        if (!STATE) Cf[q][i] = Cv[q].at(i);
      }
    if (tile + 1 < at.tile1) load(min(SSM_TT, at.len - t0 - SSM_TT));
    if (!STATE && saved) {
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = 4 * (w + W * q) + k;
          if (mine && n < N) saved[(size_t)n * E + c] = h[q][k];
        }
      saved += saved_step;
    }
    __syncthreads();
    if (rows > 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 dl = *reinterpret_cast<const f32x4*>(sd + lane * SSM_PITCH + 4 * i);
        const f32x4 ul = *reinterpret_cast<const f32x4*>(su + lane * SSM_PITCH + 4 * i);
        f32x4 yl = {0.f, 0.f, 0.f, 0.f};
        if (STATE) dsum += (dl[0] + dl[1]) + (dl[2] + dl[3]);
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          float hs[4][4];
          static_for<4>([&](auto kt) {
            constexpr int t = decltype(kt)::value;
            static_for<4>([&](auto kn) {
              constexpr int n = decltype(kn)::value;
              const float a = __builtin_amdgcn_exp2f(dl[t] * A2[q][n]);
              h[q][n] = fmaf(a, h[q][n], dpp<DPP_BCAST + 4 * t + n>(Bf[q][i]) * ul[t]);
              hs[t][n] = h[q][n];
            });
          });
          if (!STATE) ssm_dots(yl, Cf[q][i], hs);
        }
        if (!STATE) *reinterpret_cast<f32x4*>(sy + w * SSM_TILE + lane * SSM_PITCH + 4 * i) = yl;
      }
    }
    __syncthreads();
    if constexpr (!STATE) {
      const rsrc_t ry = open_rsrc(yb);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = tr + r * Split::ROWS;
        RawRow<T, V, VEC> out;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float y = xv[r][i];
#pragma unroll
          for (int j = 0; j < W; ++j) y += sy[j * SSM_TILE + (tc + i) * SSM_PITCH + row];
          out.set(i, row < rows ? y * gate[r][i] : 0.f);
        }
        store_raw<T, V, VEC>(ry, row * E + tc, row < p.L - t0, left, out);
      }
      yb += SSM_TT * (long long)E;
    }
  }

  if (!mine) return;
  const size_t rec = (size_t)at.b * (p.S - 1) + at.s;
  if (STATE && w == 0) p.dsum[rec * p.E + c] = dsum;
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = 4 * (w + W * q) + k;
      if (n >= p.N) continue;
      if (STATE)
        p.rec[(rec * p.N + n) * p.E + c] = h[q][k];
      else if (p.state_out && at.s == p.S - 1)
        p.state_out[((size_t)at.b * p.E + c) * p.N + n] = h[q][k];
    }
}

// One token of each sequence: four lanes to a channel, lane q of them the states
// 4 q .. 4 q + 3 of every 16, read and written once as 16 bytes.  The state's bytes bound
// a large batch, the launch and one round of loads a small one.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void ssm_step_kernel(Ssm p, float* state) {
  const int c = blockIdx.x * 64 + (threadIdx.x >> 2), q = threadIdx.x & 3, b = blockIdx.y;
  const bool in = c < p.E;
  const int ci = in ? c : p.E - 1, g = ci / p.Eg;
  const float x = (float)((const T*)p.x)[b * p.x_b + ci];
  float d = (float)((const T*)p.dt)[b * p.dt_b + ci] + (p.bias ? p.bias[ci] : 0.f);
  const float z = p.z ? (float)((const T*)p.z)[b * p.z_b + ci] : 0.f;
  const float skip = p.D ? p.D[ci] * x : 0.f;
  const T* B = (const T*)p.B + b * p.B_b + (long long)g * p.B_g;
  const T* C = (const T*)p.C + b * p.C_b + (long long)g * p.C_g;
  const float* A = p.A + (size_t)ci * p.N;
  float* st = state + ((size_t)b * p.E + ci) * p.N;
  if (p.softplus) d = softplus(d);
  const float u = d * x;
  float y = 0.f;
  for (int n0 = 4 * q; n0 < p.N; n0 += 16) {
    f32x4 h, a;
    float Bn[4], Cn[4];
    if constexpr (VEC) {
      h = *reinterpret_cast<const f32x4*>(st + n0);
      a = *reinterpret_cast<const f32x4*>(A + n0);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = min(n0 + k, p.N - 1);
      if constexpr (!VEC) {
        h[k] = st[n];
        a[k] = A[n];
      }
      Bn[k] = (float)B[n];
      Cn[k] = (float)C[n];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[k] = fmaf(__builtin_amdgcn_exp2f(d * (a[k] * LOG2E)), h[k], u * Bn[k]);
      if (n0 + k < p.N) y = fmaf(Cn[k], h[k], y);
    }
    if (in) {
      if constexpr (VEC) {
        *reinterpret_cast<f32x4*>(st + n0) = h;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n0 + k < p.N) st[n0 + k] = h[k];
      }
    }
  }
  y += dpp<DPP_XOR1>(y);
  y += dpp<DPP_XOR2>(y);
  if (q == 0 && in) {
    y += skip;
    if (p.z) y *= z * sigmoid(z);
    ((T*)p.y)[(size_t)b * p.E + c] = (T)y;
  }
}

template <typename T, int W, int NP, bool VEC>
hipError_t fwd_launch(const Ssm& p, hipStream_t st) {
  const int nblk = p.G * p.gblocks;
  if (p.S > 1) {
    hipLaunchKernelGGL((ssm_fwd_kernel<T, W, NP, VEC, true>), dim3(nblk * (p.S - 1) * p.batch),
                       dim3(64 * W), 0, st, p);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((ssm_fwd_kernel<T, W, NP, VEC, false>), dim3(nblk * p.S * p.batch),
                     dim3(64 * W), 0, st, p);
  return hipGetLastError();
}

template <typename T, bool VEC>
hipError_t fwd_waves(const Ssm& p, hipStream_t st) {
  switch (ssm_waves(p.N)) {
    case 1: return fwd_launch<T, 1, 1, VEC>(p, st);
    case 2: return fwd_launch<T, 2, 1, VEC>(p, st);
    case 4: return fwd_launch<T, 4, 1, VEC>(p, st);
    default:
      return ssm_passes(p.N) == 1 ? fwd_launch<T, 8, 1, VEC>(p, st) : fwd_launch<T, 8, 2, VEC>(p, st);
  }
}

// Segments of a sequence: as many as bring the waves to two a SIMD
int ssm_segments(int batch, int G, int Eg, int N, int L, bool) {
  const int tiles = (L + SSM_TT - 1) / SSM_TT;
  const long long waves = (long long)batch * G * ((Eg + SSM_CH - 1) / SSM_CH) * ssm_waves(N);
  const long long want = 8LL * device_geom().cus;
  long long s = want / waves;
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

hipError_t launch_ssm_step(const Ssm& p, float* state, bool is_bf16, hipStream_t st) {
  const dim3 grid((p.E + 63) / 64, p.batch);
  const bool vec = p.N % 4 == 0 && ((uintptr_t)state | (uintptr_t)p.A) % 16 == 0;
  if (is_bf16 && vec)
    hipLaunchKernelGGL((ssm_step_kernel<bf16, true>), grid, dim3(256), 0, st, p, state);
  else if (is_bf16)
    hipLaunchKernelGGL((ssm_step_kernel<bf16, false>), grid, dim3(256), 0, st, p, state);
  else if (vec)
    hipLaunchKernelGGL((ssm_step_kernel<float, true>), grid, dim3(256), 0, st, p, state);
  else
    hipLaunchKernelGGL((ssm_step_kernel<float, false>), grid, dim3(256), 0, st, p, state);
  return hipGetLastError();
}

}  // namespace lz
