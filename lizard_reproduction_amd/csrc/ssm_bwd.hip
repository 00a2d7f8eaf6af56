// Gradients of the selective state space scan.
//
// With s = silu(z) and dm = dy s (the gradient of sum_n C h + D x), walking back:
//   g_t[n] = dm_t C_t[n] + a_{t+1}[n] g_{t+1}[n],    v_t[n] = a_t[n] g_t[n] h_{t-1}[n]
//   du_t = sum_n g_t[n] B_t[n],                      ddelta_t = sum_n v_t[n] A[n] + x_t du_t
//   dx_t = delta_t du_t + D dm_t,                    ddt_t = ddelta_t sigmoid(dt_t + bias)
//   dB_t[n] = sum_channels g_t[n] u_t,               dC_t[n] = sum_channels dm_t h_t[n]
//   dA[n] = sum_t v_t[n] delta_t,   dD = sum_t dm_t x_t,   dbias = sum_t ddt_t
//
// The forward kept the state before each tile of 16 tokens.  A workgroup takes 64 channels
// as in the forward and walks the tiles from the last; in each it walks forward once, every
// decay and state of its 16 tokens staying in registers (128 of them), then back.  What is
// summed over n meets in LDS, the waves' shares side by side; what is summed over channels
// is added across the wave, eight sums at a time, each step halving the lanes that carry
// one (17 instructions for the 8 sums of 64 lanes), and its 64-channel shares, as the
// sequences' shares of dA, dD and dbias, go to memory for a second launch that adds them in
// order: no atomics, the same bits every time.
#include "ssm.hpp"

namespace lz {

// a + b of the two registers that a swap of a's and b's half waves (rows of 16) leaves:
// the swapped halves next to each other, each with what the other register held of it.
// (The swap's results are copied out first: a bit cast of an element of its vector reads
// element 0.)
template <bool ROWS>
__device__ __forceinline__ float swap_add(float a, float b) {
  const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
  uint32_t lo, hi;
  if constexpr (ROWS) {
    const auto s = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    lo = s[0], hi = s[1];
  } else {
    const auto s = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    lo = s[0], hi = s[1];
  }
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// The sums of v0 .. v7 over the wave: lane l gets sum l / 8.
__device__ __forceinline__ float wave_sums8(const float (&v)[8]) {
  float q[4], r[2];
#pragma unroll
  for (int k = 0; k < 4; ++k) q[k] = swap_add<false>(v[k], v[k + 4]);
#pragma unroll
  for (int k = 0; k < 2; ++k) r[k] = swap_add<true>(q[k], q[k + 2]);
  // lanes 0 - 7 of a row go on with r[0], 8 - 15 with r[1]
  const bool hi = threadIdx.x & 8;
  float s = hi ? r[1] : r[0];
  s += dpp<DPP_ROR8>(hi ? r[0] : r[1]);
  s += dpp<DPP_HALF_MIRROR>(s);
  s += dpp<DPP_XOR1>(s);
  s += dpp<DPP_XOR2>(s);
  return s;
}

// The walk of both backward kernels over a segment: with STATE only the carried gradient,
// to rec, and the sum of delta, for the segments but the first.
template <typename T, int W, int NP, bool VEC, bool STATE>
__global__ __launch_bounds__(64 * W, W == 8 ? 2 : W == 4 ? 2 : 1) void ssm_bwd_kernel(Ssm p, SsmGrad gr) {
  using Split = SsmSplit<W>;
  constexpr int V = Split::V, R = Split::R;
  extern __shared__ float lds[];
  float* const sd = lds;                    // delta
  float* const su = sd + SSM_TILE;          // delta x
  float* const sg = su + SSM_TILE;          // dm
  float* const pu = sg + SSM_TILE;          // [W]: the waves' shares of du,
  float* const pd = pu + W * SSM_TILE;      // of sum_n v A
  float* const py = pd + W * SSM_TILE;      // and of sum_n C h
  const int segments = STATE ? p.S - 1 : p.S;
  SsmPlace at(p, segments);
  if constexpr (STATE) {   // segments 1 .. S - 1
    ++at.s;
    at.tile0 = at.s * p.seg_tiles;
    at.tile1 = min(p.tiles, at.tile0 + p.seg_tiles);
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = at.c0 + lane;
  const bool mine = lane < at.cols;
  const int N = p.N, E = p.E;

  float A2[NP][4], carry[NP][4], dA[NP][4];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int n = 4 * (w + W * q) + k;
      A2[q][k] = mine && n < N ? p.A[(size_t)c * N + n] * LOG2E : 0.f;
      carry[q][k] = dA[q][k] = 0.f;
    }
  if constexpr (!STATE) {
    // what the later segments carry back
    for (int j = p.S - 1; j > at.s; --j) {
      const size_t rec = (size_t)at.b * (p.S - 1) + j - 1;
      const float d = mine ? gr.dsum[rec * E + c] : 0.f;
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = 4 * (w + W * q) + k;
          if (mine && n < N)
            carry[q][k] = fmaf(__builtin_amdgcn_exp2f(A2[q][k] * d), carry[q][k],
                               gr.rec[(rec * N + n) * E + c]);
        }
    }
  }

  const int tr = tid / Split::COLS, tc = (tid % Split::COLS) * V, left = at.cols - tc;
  float bias[V], D[V], dD[V], dbias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = p.bias && i < left ? p.bias[at.c0 + tc + i] : 0.f;
    D[i] = p.D && i < left ? p.D[at.c0 + tc + i] : 0.f;
    dD[i] = dbias[i] = 0.f;
  }
  const long long last = (long long)(at.tile1 - 1) * SSM_TT;
  const int x_t = p.x_t, dt_t = p.dt_t, z_t = p.z_t, B_t = p.B_t, C_t = p.C_t;
  const bool has_z = p.z, soft = p.softplus;
  const T* xb = (const T*)p.x + at.b * p.x_b + last * x_t + at.c0;
  const T* db = (const T*)p.dt + at.b * p.dt_b + last * dt_t + at.c0;
  const T* zb = has_z ? (const T*)p.z + at.b * p.z_b + last * z_t + at.c0 : nullptr;
  const T* Bb = (const T*)p.B + at.b * p.B_b + last * B_t + (long long)at.g * p.B_g;
  const T* Cb = (const T*)p.C + at.b * p.C_b + last * C_t + (long long)at.g * p.C_g;
  long long yo = ((long long)at.b * p.L + last) * E + at.c0;   // rows of dy, next to load
  const T* dyb = (const T*)gr.dy + yo;
  const float* saved = p.saved + ((size_t)at.b * p.tiles + at.tile1 - 1) * N * E + c;
  const int NQ = 4 * W * NP;
  float* bc = STATE ? nullptr
                    : gr.part_bc + (((long long)at.blk * p.batch + at.b) * p.L + last) * 2 * NQ;

  RawRow<T, V, VEC> xr[R], dr[R], zr[R], yr[R];
  SsmVec<T> Bv[NP], Cv[NP];
  float h0[NP][4];
  auto load = [&](int rows) {
    const rsrc_t rx = open_rsrc(xb), rd = open_rsrc(db), rz = open_rsrc(zb), ry = open_rsrc(dyb);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = tr + r * Split::ROWS;
      xr[r] = load_raw<T, V, VEC>(rx, row * x_t + tc, row < rows, left);
      dr[r] = load_raw<T, V, VEC>(rd, row * dt_t + tc, row < rows, left);
      zr[r] = load_raw<T, V, VEC>(rz, row * z_t + tc, has_z && row < rows, left);
      yr[r] = load_raw<T, V, VEC>(ry, row * E + tc, row < rows, left);
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      if (!STATE) Bv[q].load(Bb, rows, B_t, N, 4 * (w + W * q), lane);
      Cv[q].load(Cb, rows, C_t, N, 4 * (w + W * q), lane);
      if (!STATE) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = 4 * (w + W * q) + k;
          h0[q][k] = mine && n < N ? saved[(size_t)n * E] : 0.f;
        }
      }
    }
    xb -= SSM_TT * (long long)x_t;
    db -= SSM_TT * (long long)dt_t;
    if (has_z) zb -= SSM_TT * (long long)z_t;
    dyb -= SSM_TT * (long long)E;
    Bb -= SSM_TT * (long long)B_t;
    Cb -= SSM_TT * (long long)C_t;
    saved -= (size_t)N * E;
  };

  float dsum = 0.f;
  load(min(SSM_TT, p.L - (int)last));
  for (int tile = at.tile1 - 1; tile >= at.tile0; --tile) {
    const int t0 = tile * SSM_TT;
    const int rows = min(SSM_TT, p.L - t0);
    float xv[R][V], dl[R][V], sl[R][V], zv[R][V], dyv[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = tr + r * Split::ROWS;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = xr[r].at(i), pre = dr[r].at(i) + bias[i], z = zr[r].at(i);
        const float dy = yr[r].at(i);
        const float d = row < rows ? soft ? softplus(pre) : pre : 0.f;
        const float dm = has_z ? dy * (z * sigmoid(z)) : dy;
        sd[(tc + i) * SSM_PITCH + row] = d;
        sg[(tc + i) * SSM_PITCH + row] = dm;
        if (!STATE) su[(tc + i) * SSM_PITCH + row] = d * x;
        xv[r][i] = x, dl[r][i] = d, sl[r][i] = soft ? sigmoid(pre) : 1.f;
        zv[r][i] = z, dyv[r][i] = dy;
      }
    }
    float Bf[NP][4], Cf[NP][4], hb[NP][4];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!STATE) Bf[q][i] = Bv[q].at(i);
        Cf[q][i] = Cv[q].at(i);
        if (!STATE) hb[q][i] = h0[q][i];
      }
    if (tile > at.tile0) load(SSM_TT);
    __syncthreads();
    if constexpr (STATE) {
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + lane * SSM_PITCH + 4 * i);
        const f32x4 g4 = *reinterpret_cast<const f32x4*>(sg + lane * SSM_PITCH + 4 * i);
        dsum += (d4[0] + d4[1]) + (d4[2] + d4[3]);
        static_for<4>([&](auto kt) {
          constexpr int t = 3 - decltype(kt)::value;
#pragma unroll
          for (int q = 0; q < NP; ++q)
            static_for<4>([&](auto kn) {
              constexpr int n = decltype(kn)::value;
              carry[q][n] = __builtin_amdgcn_exp2f(d4[t] * A2[q][n]) *
                            (dpp<DPP_BCAST + 4 * t + n>(Cf[q][i]) * g4[t] + carry[q][n]);
            });
        });
      }
    } else {
      float bcsum[NP][2];
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        float a[16][4], h[16][4];
        // forward over the tile
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + lane * SSM_PITCH + 4 * i);
          const f32x4 u4 = *reinterpret_cast<const f32x4*>(su + lane * SSM_PITCH + 4 * i);
          float hs[4][4];
          static_for<4>([&](auto kt) {
            constexpr int t = decltype(kt)::value;
            static_for<4>([&](auto kn) {
              constexpr int n = decltype(kn)::value;
              const float before = 4 * i + t ? h[(4 * i + t + 15) % 16][n] : hb[q][n];
              a[4 * i + t][n] = __builtin_amdgcn_exp2f(d4[t] * A2[q][n]);
              h[4 * i + t][n] = fmaf(a[4 * i + t][n], before,
                                     dpp<DPP_BCAST + 4 * t + n>(Bf[q][i]) * u4[t]);
              hs[t][n] = h[4 * i + t][n];
            });
          });
          if (has_z) {
            float* to = py + w * SSM_TILE + lane * SSM_PITCH + 4 * i;
            f32x4 yl = {0.f, 0.f, 0.f, 0.f};
            if (q) yl = *reinterpret_cast<const f32x4*>(to);
            ssm_dots(yl, Cf[q][i], hs);
            *reinterpret_cast<f32x4*>(to) = yl;
          }
        }
        // and back
        bcsum[q][0] = bcsum[q][1] = 0.f;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + lane * SSM_PITCH + 4 * i);
          const f32x4 u4 = *reinterpret_cast<const f32x4*>(su + lane * SSM_PITCH + 4 * i);
          const f32x4 g4 = *reinterpret_cast<const f32x4*>(sg + lane * SSM_PITCH + 4 * i);
          float gs[4][4];
          f32x4 dv = {0.f, 0.f, 0.f, 0.f}, du = {0.f, 0.f, 0.f, 0.f};
          float* const tu = pu + w * SSM_TILE + lane * SSM_PITCH + 4 * i;
          float* const td = pd + w * SSM_TILE + lane * SSM_PITCH + 4 * i;
          if (q) {
            dv = *reinterpret_cast<const f32x4*>(td);
            du = *reinterpret_cast<const f32x4*>(tu);
          }
          static_for<4>([&](auto kt) {
            constexpr int t = 3 - decltype(kt)::value;
            const int tt = 4 * i + t;
            float v8[8];
            static_for<4>([&](auto kn) {
              constexpr int n = decltype(kn)::value;
              const float g = dpp<DPP_BCAST + 4 * t + n>(Cf[q][i]) * g4[t] + carry[q][n];
              gs[t][n] = g;
              v8[n] = g * u4[t];
              v8[4 + n] = g4[t] * h[tt][n];
              carry[q][n] = a[tt][n] * g;
              const float v = carry[q][n] * (tt ? h[(tt + 15) % 16][n] : hb[q][n]);
              dv[t] = fmaf(v, A2[q][n], dv[t]);
              dA[q][n] = fmaf(v, d4[t], dA[q][n]);
            });
            const float s8 = wave_sums8(v8);
            if ((lane & 7) == (tt & 7)) bcsum[q][tt >> 3] = s8;
          });
          ssm_dots(du, Bf[q][i], gs);
          *reinterpret_cast<f32x4*>(td) = dv;
          *reinterpret_cast<f32x4*>(tu) = du;
        }
        // lane l: of token l % 8 (+ 8), B's (l < 32) or C's sum for state (l / 8) % 4
        const rsrc_t rb = open_rsrc(bc);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int row = 8 * k + (lane & 7), idx = lane >> 3;
          const uint32_t off =
              (uint32_t)((2 * row + (idx >> 2)) * NQ + 4 * (w + W * q) + (idx & 3)) * 4u;
          __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, bcsum[q][k]), rb,
                                                row < rows ? off : OOB, 0, 0);
        }
      }
      bc -= SSM_TT * 2 * NQ;
    }
    __syncthreads();
    if constexpr (!STATE) {
      const long long o = ((long long)at.b * p.L + t0) * E + at.c0;
      const rsrc_t rx = open_rsrc((T*)gr.dx + o), rd = open_rsrc((T*)gr.ddt + o);
      const rsrc_t rz = open_rsrc(has_z ? (T*)gr.dz + o : nullptr);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = tr + r * Split::ROWS;
        RawRow<T, V, VEC> ox, od, oz;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int e = (tc + i) * SSM_PITCH + row;
          float du = 0.f, dv = 0.f, y = xv[r][i] * D[i];
#pragma unroll
          for (int j = 0; j < W; ++j) {
            du += pu[j * SSM_TILE + e];
            dv += pd[j * SSM_TILE + e];
            if (has_z) y += py[j * SSM_TILE + e];
          }
          const float z = zv[r][i], sz = sigmoid(z), dy = dyv[r][i];
          const float dm = has_z ? dy * (z * sz) : dy;
          const float ddt = fmaf(xv[r][i], du, dv * LN2) * sl[r][i];
          ox.set(i, fmaf(dl[r][i], du, D[i] * dm));
          od.set(i, ddt);
          if (has_z) oz.set(i, dy * y * (sz * (1.f + z * (1.f - sz))));
          if (row < rows && i < left) {
            dD[i] += dm * xv[r][i];
            dbias[i] += ddt;
          }
        }
        store_raw<T, V, VEC>(rx, row * E + tc, row < rows, left, ox);
        store_raw<T, V, VEC>(rd, row * E + tc, row < rows, left, od);
        if (has_z) store_raw<T, V, VEC>(rz, row * E + tc, row < rows, left, oz);
      }
    }
  }

  if constexpr (STATE) {
    if (!mine) return;
    const size_t rec = (size_t)at.b * (p.S - 1) + at.s - 1;
    if (w == 0) gr.dsum[rec * E + c] = dsum;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = 4 * (w + W * q) + k;
        if (n < N) gr.rec[(rec * N + n) * E + c] = carry[q][k];
      }
  } else {
    const size_t part = (size_t)at.b * p.S + at.s;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = 4 * (w + W * q) + k;
        if (mine && n < N) gr.part_a[(part * N + n) * E + c] = dA[q][k];
      }
    // the rows' shares of dD and dbias meet in LDS (the delta and u tiles)
    __syncthreads();
    float* const red = lds;   // [2][ROWS][64]
#pragma unroll
    for (int i = 0; i < V; ++i) {
      red[tr * SSM_CH + tc + i] = dD[i];
      red[(Split::ROWS + tr) * SSM_CH + tc + i] = dbias[i];
    }
    __syncthreads();
    for (int i = tid; i < 2 * SSM_CH; i += 64 * W) {
      const int which = i / SSM_CH, ch = i % SSM_CH;
      float sum = 0.f;
      for (int r = 0; r < Split::ROWS; ++r) sum += red[(which * Split::ROWS + r) * SSM_CH + ch];
      if (ch < at.cols) gr.part_d[(part * 2 + which) * E + at.c0 + ch] = sum;
    }
  }
}

template <typename T, int W, int NP, bool VEC>
hipError_t bwd_launch(const Ssm& p, const SsmGrad& gr, hipStream_t st) {
  const int nblk = p.G * p.gblocks;
  if (p.S > 1) {
    constexpr int bytes = 3 * SSM_TILE * 4;
    hipLaunchKernelGGL((ssm_bwd_kernel<T, W, NP, VEC, true>), dim3(nblk * (p.S - 1) * p.batch),
                       dim3(64 * W), bytes, st, p, gr);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  constexpr int bytes = (3 + 3 * W) * SSM_TILE * 4;
  if (hipError_t e = ensure_lds<ssm_bwd_kernel<T, W, NP, VEC, false>>(bytes); e != hipSuccess) return e;
  hipLaunchKernelGGL((ssm_bwd_kernel<T, W, NP, VEC, false>), dim3(nblk * p.S * p.batch),
                     dim3(64 * W), bytes, st, p, gr);
  return hipGetLastError();
}

template <typename T, bool VEC>
hipError_t bwd_waves(const Ssm& p, const SsmGrad& gr, hipStream_t st) {
  switch (ssm_waves(p.N)) {
    case 1: return bwd_launch<T, 1, 1, VEC>(p, gr, st);
    case 2: return bwd_launch<T, 2, 1, VEC>(p, gr, st);
    case 4: return bwd_launch<T, 4, 1, VEC>(p, gr, st);
    default:
      return ssm_passes(p.N) == 1 ? bwd_launch<T, 8, 1, VEC>(p, gr, st)
                                  : bwd_launch<T, 8, 2, VEC>(p, gr, st);
  }
}

hipError_t launch_ssm_bwd(const Ssm& p, const SsmGrad& gr, void* dB, void* dC, float* dA,
                          float* dD, float* dbias, bool is_bf16, bool vec, hipStream_t st) {
  hipError_t e = is_bf16 ? vec ? bwd_waves<bf16, true>(p, gr, st) : bwd_waves<bf16, false>(p, gr, st)
                 : vec   ? bwd_waves<float, true>(p, gr, st)
                         : bwd_waves<float, false>(p, gr, st);
  if (e != hipSuccess) return e;
  const int NQ = 4 * ssm_waves(p.N) * ssm_passes(p.N), parts = p.batch * p.S;
  const long long rows = (long long)p.batch * p.L;
  // dB and dC: the blocks of a group, for each group
  for (int g0 = 0; g0 < p.G; g0 += SUM_JOBS / 2) {
    SumJobs jobs = {};
    for (int g = g0; g < p.G && g < g0 + SUM_JOBS / 2; ++g)
      for (int k = 0; k < 2; ++k) {
        SumJob& j = jobs.job[jobs.n++];
        j.src = gr.part_bc + (long long)g * p.gblocks * rows * 2 * NQ + k * NQ;
        void* const dst = k ? dC : dB;
        j.dst = is_bf16 ? (void*)((bf16*)dst + g * p.N) : (void*)((float*)dst + g * p.N);
        j.part_stride = rows * 2 * NQ;
        j.row_stride = 2 * NQ;
        j.out_row = (long long)p.G * p.N;
        j.out_col = 1;
        j.rows = (int)rows, j.cols = p.N, j.parts = p.gblocks, j.bf16 = is_bf16;
      }
    if (e = launch_sums(jobs, st); e != hipSuccess) return e;
  }
  SumJobs jobs = {};
  jobs.job[jobs.n++] = SumJob{gr.part_a, dA, (long long)p.N * p.E, p.E, 1, p.N, p.N, p.E, parts, 0};
  for (int k = 0; k < 2; ++k)
    if (float* dst = k ? dbias : dD)
      jobs.job[jobs.n++] =
          SumJob{gr.part_d + k * (long long)p.E, dst, 2LL * p.E, 0, 0, 1, 1, p.E, parts, 0};
  return launch_sums(jobs, st);
}

}  // namespace lz
