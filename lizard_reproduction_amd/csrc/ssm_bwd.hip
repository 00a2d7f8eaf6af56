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
// decay and state of its 16 tokens staying in registers, then back.  What is
// summed over n meets in LDS, the waves' shares side by side; what is summed over channels
// is added across the wave, four tokens' sixteen sums at a time, and its 64-channel shares, as
// the sequences' shares of dA, dD and dbias, go to memory for a second launch that adds them
// in order: no atomics, the same bits every time.  More than 16 states are taken 16 a launch
// (in one, a wave's registers did not hold them: N = 24 took 2.8 times as long as 16).
//
// The vector units bound it: B = 4, L = 2048, E = 4096, N = 16 in bf16 takes 435 us, 94 % of
// them busy, a little over half with the twelve instructions and the exponential that each
// (token, channel, n) takes.  (The sums over channels on the matrix units, 16 x 16 x 4 in
// fp32: 470 -> 678 us, as their operands have to be laid out across lanes.  A helper's rows
// kept by turns instead of copied: 3 % slower.)
#include "ssm.hpp"

namespace lz {

// The sums over the wave of v[0] .. v[15], each step halving the registers that carry them:
// two values share a row of 16 lanes by its halves, four by its quads (a lane operand's sum
// written to some banks of four lanes only, which takes no select: written out, with two
// instructions at least from a register's write to its use as such an operand), then 8 and
// 16 the wave by its rows.  Lane l gets v[4 (l / 16) + 2 (l / 4 % 2) + l / 8 % 2].  (36 issue
// slots; by swaps and selects from the start, eight values at a time, 50.)
__device__ __forceinline__ float wave_sums16(float (&v)[16]) {
#define LZ_R8(d, s, m) "v_add_f32_dpp %" #d ", %" #s ", %" #s " row_ror:8 row_mask:0xf bank_mask:" #m "\n"
#define LZ_HM(d, s, m) \
  "v_add_f32_dpp %" #d ", %" #s ", %" #s " row_half_mirror row_mask:0xf bank_mask:" #m "\n"
  asm("s_nop 1\n"
      LZ_R8(0, 0, 0xf) LZ_R8(1, 1, 0xf) LZ_R8(2, 2, 0xf) LZ_R8(3, 3, 0xf)
      LZ_R8(4, 4, 0xf) LZ_R8(5, 5, 0xf) LZ_R8(6, 6, 0xf) LZ_R8(7, 7, 0xf)
      LZ_R8(0, 8, 0xc) LZ_R8(1, 9, 0xc) LZ_R8(2, 10, 0xc) LZ_R8(3, 11, 0xc)
      LZ_R8(4, 12, 0xc) LZ_R8(5, 13, 0xc) LZ_R8(6, 14, 0xc) LZ_R8(7, 15, 0xc)
      LZ_HM(0, 0, 0xf) LZ_HM(2, 2, 0xf) LZ_HM(4, 4, 0xf) LZ_HM(6, 6, 0xf)
      LZ_HM(0, 1, 0xa) LZ_HM(2, 3, 0xa) LZ_HM(4, 5, 0xa) LZ_HM(6, 7, 0xa)
      : "+&v"(v[0]), "+&v"(v[2]), "+&v"(v[4]), "+&v"(v[6]), "+&v"(v[8]), "+&v"(v[10]),
        "+&v"(v[12]), "+&v"(v[14])
      : "v"(v[1]), "v"(v[3]), "v"(v[5]), "v"(v[7]), "v"(v[9]), "v"(v[11]), "v"(v[13]), "v"(v[15]));
#undef LZ_R8
#undef LZ_HM
  float s = swap_add<true>(swap_add<false>(v[0], v[8]), swap_add<false>(v[4], v[12]));
  s += dpp<DPP_XOR1>(s);
  s += dpp<DPP_XOR2>(s);
  return s;
}

// STATE: the gradient that a segment carries back alone, and its sum of delta, for the
// segments but the first.
template <int W, bool STATE>
constexpr int ssm_bwd_lds() {   // tiles, two of each
  return 2 * (STATE ? 2 : 3 + 2 * W);
}

template <typename T, int W, bool VEC, bool STATE>
__global__ __launch_bounds__(64 * (W + SSM_HELPERS), W == 8 ? 3 : 2) void ssm_bwd_kernel(Ssm p, SsmGrad gr) {
  constexpr int V = SSM_V;
  extern __shared__ float lds[];
  auto sd = [&](int buf) { return lds + buf * SSM_TILE; };              // delta
  auto sg = [&](int buf) { return lds + (2 + buf) * SSM_TILE; };      // dm
  auto su = [&](int buf) { return lds + (4 + buf) * SSM_TILE; };  // delta x
  // the waves' shares of du and of sum_n v A
  auto pu = [&](int buf, int j) { return lds + ((3 + j) * 2 + buf) * SSM_TILE; };
  auto pd = [&](int buf, int j) { return lds + ((3 + W + j) * 2 + buf) * SSM_TILE; };
  const int segments = STATE ? p.S - 1 : p.S;
  SsmPlace at(p, segments);
  if constexpr (STATE) {   // segments 1 .. S - 1
    ++at.s;
    at.tile0 = at.s * p.seg_tiles;
    at.tile1 = min(p.tiles, at.tile0 + p.seg_tiles);
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int E = p.E, N = p.N;
  const bool has_z = p.z, soft = p.softplus;
  const long long last = (long long)(at.tile1 - 1) * SSM_TT;
  auto rows_of = [&](int tile) { return min(SSM_TT, p.L - tile * SSM_TT); };

  // --- rows to delta, u and dm; the waves' shares to gradients (helper) ------------------
  const int tid = (int)threadIdx.x - 64 * W;
  const int row = tid / SSM_COLS, tc = (tid % SSM_COLS) * V, left = at.cols - tc;
  float bias[V], D[V], dD[V], dbias[V];
  const int x_t = p.x_t, dt_t = p.dt_t, z_t = p.z_t;
  const T* xb = (const T*)p.x + at.b * p.x_b + last * x_t + at.c0;
  const T* db = (const T*)p.dt + at.b * p.dt_b + last * dt_t + at.c0;
  const T* zb = has_z ? (const T*)p.z + at.b * p.z_b + last * z_t + at.c0 : nullptr;
  const T* dyb = (const T*)gr.dy + ((long long)at.b * p.L + last) * E + at.c0;
  const float* mb = p.mixed + ((long long)at.b * p.L + last) * E + at.c0;
  struct Rows {   // of a tile
    RawRow<T, V, VEC> x, dt, z, dy;
    RawRow<float, V, VEC> mixed;
  };
  struct Kept {   // of a tile, from its beginning to its end
    float x[V], delta[V], dm[V], slope[V], dz[V];
  };
  auto load_params = [&] {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      bias[i] = p.bias && i < left ? p.bias[at.c0 + tc + i] : 0.f;
      D[i] = p.D && i < left ? p.D[at.c0 + tc + i] : 0.f;
      dD[i] = dbias[i] = 0.f;
    }
  };
  auto load_rows = [&](int rows, Rows& r) {
    const bool in = row < rows;
    if (!STATE) r.x = load_raw<T, V, VEC>(open_rsrc(xb), row * x_t + tc, in, left);
    r.dt = load_raw<T, V, VEC>(open_rsrc(db), row * dt_t + tc, in, left);
    r.z = load_raw<T, V, VEC>(open_rsrc(zb), row * z_t + tc, has_z && in, left);
    r.dy = load_raw<T, V, VEC>(open_rsrc(dyb), row * E + tc, in, left);
    if (!STATE) {
      r.mixed = load_raw<float, V, VEC>(open_rsrc(mb), row * E + tc, has_z && in, left);
      mb -= SSM_TT * (long long)E;
    }
    xb -= SSM_TT * (long long)x_t;
    db -= SSM_TT * (long long)dt_t;
    if (has_z) zb -= SSM_TT * (long long)z_t;
    dyb -= SSM_TT * (long long)E;
  };
  auto prep = [&](int rows, int buf, const Rows& r, Kept& k) {
    const int e = row * SSM_CH + tc;
    float u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float pre = r.dt.at(i) + bias[i];
      k.delta[i] = pre, k.slope[i] = 1.f;
      if (soft) k.delta[i] = STATE ? softplus(pre) : softplus_slope(pre, k.slope[i]);
      k.dm[i] = r.dy.at(i);
      if (!STATE) k.x[i] = r.x.at(i);
    }
    if (has_z) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = r.z.at(i), s = sigmoid(z), dy = k.dm[i], zs = z * s;
        k.dm[i] = dy * zs;
        if (!STATE) k.dz[i] = dy * r.mixed.at(i) * fmaf(zs, 1.f - s, s);
      }
    }
    if (rows < SSM_TT && row >= rows) {
#pragma unroll
      for (int i = 0; i < V; ++i) k.delta[i] = 0.f;
    }
    put_row(sd(buf) + e, k.delta);
    put_row(sg(buf) + e, k.dm);
    if (!STATE) {
#pragma unroll
      for (int i = 0; i < V; ++i) u[i] = k.delta[i] * k.x[i];
      put_row(su(buf) + e, u);
    }
  };
  auto finish = [&](int tile, int buf, const Kept& k) {
    const int rows = rows_of(tile), e = row * SSM_CH + tc;
    const long long o = ((long long)at.b * p.L + (long long)tile * SSM_TT) * E + at.c0;
    const uint32_t off = row * E + tc;
    const bool in = row < rows;
    float sum[2][V];   // of du and of sum_n v A
#pragma unroll
    for (int i = 0; i < V; ++i) sum[0][i] = sum[1][i] = 0.f;
    if (!gr.first) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const auto r = load_raw<float, V, VEC>(open_rsrc(gr.acc + j * gr.acc_step + o), off, in, left);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[j][i] = r.at(i);
      }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
      add_row(sum[0], pu(buf, j) + e);
      add_row(sum[1], pd(buf, j) + e);
    }
    if (!gr.last) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        RawRow<float, V, VEC> r;
        r.pack(sum[j]);
        store_raw<float, V, VEC>(open_rsrc(gr.acc + j * gr.acc_step + o), off, in, left, r);
      }
      return;
    }
    RawRow<T, V, VEC> ox, od, oz;
    float dx[V], ddts[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float ddt = fmaf(k.x[i], sum[0][i], sum[1][i] * LN2) * k.slope[i];
      dx[i] = fmaf(k.delta[i], sum[0][i], D[i] * k.dm[i]);
      ddts[i] = ddt;
      dD[i] = fmaf(k.dm[i], k.x[i], dD[i]);   // x and dy are zero where there is no row
      if (in && i < left) dbias[i] += ddt;
    }
    ox.pack(dx), od.pack(ddts);
    store_raw<T, V, VEC>(open_rsrc((T*)gr.dx + o), off, in, left, ox);
    store_raw<T, V, VEC>(open_rsrc((T*)gr.ddt + o), off, in, left, od);
    if (has_z) {
      oz.pack(k.dz);
      store_raw<T, V, VEC>(open_rsrc((T*)gr.dz + o), off, in, left, oz);
    }
  };

  // --- the walk (scan) --------------------------------------------------------------------
  const int w = wave, c = at.c0 + lane, n0 = gr.n0 + 2 * w;
  const bool mine = lane < at.cols;
  const int B_t = p.B_t, C_t = p.C_t;
  const T* Bb = (const T*)p.B + at.b * p.B_b + last * B_t + (long long)at.g * p.B_g;
  const T* Cb = (const T*)p.C + at.b * p.C_b + last * C_t + (long long)at.g * p.C_g;
  const float* saved = p.saved + ((size_t)at.b * p.tiles + at.tile1 - 1) * N * E + c;
  float* bc = STATE ? nullptr
                    : gr.part_bc + (((long long)at.blk * p.batch + at.b) * p.L + last) * 2 * gr.NQ;
  const int NQ = gr.NQ;
  float A2[2], carry[2], dA[2], dsum = 0.f;
  SsmVec<T, 2> Bv, Cv;
  float h0[2];
  auto start = [&] {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = n0 + k;
      A2[k] = mine && n < N ? p.A[(size_t)c * N + n] * LOG2E : 0.f;
      carry[k] = dA[k] = 0.f;
    }
    if constexpr (!STATE) {
      // what the later segments carry back
      for (int j = p.S - 1; j > at.s; --j) {
        const size_t rec = (size_t)at.b * (p.S - 1) + j - 1;
        const float d = mine ? gr.dsum[rec * E + c] : 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int n = n0 + k;
          if (mine && n < N)
            carry[k] = fmaf(__builtin_amdgcn_exp2f(A2[k] * d), carry[k],
                            gr.rec[(rec * N + n) * E + c]);
        }
      }
    }
  };
  auto load_bc = [&](int rows) {
    if (!STATE) Bv.load(Bb, rows, B_t, N, n0, lane);
    Cv.load(Cb, rows, C_t, N, n0, lane);
    if (!STATE) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int n = n0 + k;
        h0[k] = mine && n < N ? saved[(size_t)n * E] : 0.f;
      }
    }
  };
  auto next_bc = [&] {
    Bb -= SSM_TT * (long long)B_t;
    Cb -= SSM_TT * (long long)C_t;
    saved -= (size_t)N * E;
  };
  auto scan_state = [&](int buf) {
    const float Cf[2] = {Cv.at(0), Cv.at(1)};
    static_for<4>([&](auto ki) {
      constexpr int i = 3 - decltype(ki)::value;
      const f32x4 d4 = get_tokens(sd(buf), 4 * i, lane), g4 = get_tokens(sg(buf), 4 * i, lane);
      dsum += (d4[0] + d4[1]) + (d4[2] + d4[3]);
      static_for<4>([&](auto kt) {
        constexpr int t = 3 - decltype(kt)::value;
        float g[2];
        ssm_fma2<8 * (i & 1) + 2 * t>(g, Cf[i >> 1], g4[t], carry);
#pragma unroll
        for (int n = 0; n < 2; ++n) carry[n] = __builtin_amdgcn_exp2f(d4[t] * A2[n]) * g[n];
      });
    });
  };
  auto scan = [&](int tile, int buf, bool more) {
    const int rows = rows_of(tile);
    const float Bf[2] = {Bv.at(0), Bv.at(1)}, Cf[2] = {Cv.at(0), Cv.at(1)}, hb[2] = {h0[0], h0[1]};
    float a[16][2], h[16][2], bcsum = 0.f;
    if (more) load_bc(SSM_TT);
    // forward over the tile
    static_for<16>([&](auto kt) {
      constexpr int tt = decltype(kt)::value;
      const float d = sd(buf)[tt * SSM_CH + lane], u = su(buf)[tt * SSM_CH + lane];
      static_for<2>([&](auto kn) {
        constexpr int n = decltype(kn)::value;
        a[tt][n] = __builtin_amdgcn_exp2f(d * A2[n]);
        h[tt][n] = fmaf(a[tt][n], tt ? h[(tt + 15) % 16][n] : hb[n],
                        dpp<DPP_BCAST + 2 * (tt & 7) + n>(Bf[tt >> 3]) * u);
      });
    });
    // and back
    static_for<4>([&](auto ki) {
      constexpr int i = 3 - decltype(ki)::value, K = 8 * (i & 1);
      const f32x4 d4 = get_tokens(sd(buf), 4 * i, lane), u4 = get_tokens(su(buf), 4 * i, lane);
      const f32x4 g4 = get_tokens(sg(buf), 4 * i, lane);
      float gs[4][2], bc16[16];
      f32x4 dv = {0.f, 0.f, 0.f, 0.f}, du;
      static_for<4>([&](auto kt) {
        constexpr int t = 3 - decltype(kt)::value, tt = 4 * i + t;
        ssm_fma2<K + 2 * t>(gs[t], Cf[i >> 1], g4[t], carry);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float g = gs[t][n];
          bc16[4 * t + n] = g * u4[t];
          bc16[4 * t + 2 + n] = g4[t] * h[tt][n];
          carry[n] = a[tt][n] * g;
          const float v = carry[n] * (tt ? h[(tt + 15) % 16][n] : hb[n]);
          dv[t] = fmaf(v, A2[n], dv[t]);
          dA[n] = fmaf(v, d4[t], dA[n]);
        }
      });
      const float s = wave_sums16(bc16);
      if ((lane & 3) == i) bcsum = s;
      ssm_dots<K, false>(du, Bf[i >> 1], gs);
      put_tokens(pd(buf, w), 4 * i, lane, dv);
      put_tokens(pu(buf, w), 4 * i, lane, du);
    });
    // lane l: of token 4 (l % 4) + l / 16, B's or C's (l / 4 % 2), state l / 8 % 2
    const int tk = 4 * (lane & 3) + (lane >> 4);
    const uint32_t off = (uint32_t)((2 * tk + (lane >> 2 & 1)) * NQ + n0 + (lane >> 3 & 1)) * 4u;
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, bcsum), open_rsrc(bc),
                                          tk < rows ? off : OOB, 0, 0);
    bc -= SSM_TT * 2 * NQ;
  };
  auto end = [&] {
    if (!mine) return;
    const size_t rec = (size_t)at.b * (p.S - 1) + at.s - 1, part = (size_t)at.b * p.S + at.s;
    if (STATE && w == 0) gr.dsum[rec * E + c] = dsum;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = n0 + k;
      if (n >= N) continue;
      if (STATE) gr.rec[(rec * N + n) * E + c] = carry[k];
      else gr.part_a[(part * N + n) * E + c] = dA[k];
    }
  };

  const int t0 = at.tile0, t1 = at.tile1;   // t0 < t1
  if (wave >= W) {
    // as in the forward, from the last tile on; fp32 rows one tile ahead, as two with their
    // registers spilled (training B = 2, L = 777, E = 1040, N = 24: 154 against 139 us)
    constexpr int AHEAD = IS_BF16<T> ? 2 : 1;
    Rows even, odd;
    Kept now, last, before;
    load_params();
    load_rows(rows_of(t1 - 1), even);
    if (AHEAD == 2 && t1 - 2 >= t0) load_rows(SSM_TT, odd);
    prep(rows_of(t1 - 1), 0, even, now);
    if (t1 - 1 - AHEAD >= t0) load_rows(SSM_TT, even);
    __syncthreads();
    auto step = [&](int tile, int buf, Rows& next) {
      before = now;
      if (tile > t0) {
        prep(SSM_TT, buf ^ 1, next, now);
        if (tile - 1 - AHEAD >= t0) load_rows(SSM_TT, next);
      }
      if (!STATE && tile < t1 - 1) finish(tile + 1, buf ^ 1, last);
      last = before;
      __syncthreads();
    };
    for (int tile = t1 - 1; tile >= t0; tile -= 2) {
      step(tile, 0, AHEAD == 2 ? odd : even);
      if (tile > t0) step(tile - 1, 1, even);
    }
    if (!STATE) finish(t0, (t1 - 1 - t0) & 1, last);
  } else {
    load_bc(rows_of(t1 - 1));
    next_bc();
    start();
    __syncthreads();
    for (int tile = t1 - 1; tile >= t0; --tile) {
      const int buf = (t1 - 1 - tile) & 1;
      if constexpr (STATE) {
        scan_state(buf);
        if (tile > t0) load_bc(SSM_TT);
      } else {
        scan(tile, buf, tile > t0);
      }
      next_bc();
      __syncthreads();
    }
    end();
  }
  if (!STATE && gr.last) {
    // the rows' shares of dD and dbias meet in LDS
    const size_t part = (size_t)at.b * p.S + at.s;
    __syncthreads();
    float* const red = lds;   // [2][ROWS][64]
    if (wave >= W) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        red[row * SSM_CH + tc + i] = dD[i];
        red[(SSM_ROWS + row) * SSM_CH + tc + i] = dbias[i];
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * SSM_CH; i += blockDim.x) {
      const int which = i / SSM_CH, ch = i % SSM_CH;
      float sum = 0.f;
      for (int r = 0; r < SSM_ROWS; ++r) sum += red[(which * SSM_ROWS + r) * SSM_CH + ch];
      if (ch < at.cols) gr.part_d[(part * 2 + which) * E + at.c0 + ch] = sum;
    }
  }
}

template <typename T, int W, bool VEC>
hipError_t bwd_launch(const Ssm& p, const SsmGrad& gr, hipStream_t st) {
  const int nblk = p.G * p.gblocks;
  const dim3 block(64 * (W + SSM_HELPERS));
  if (p.S > 1) {
    constexpr int bytes = ssm_bwd_lds<W, true>() * SSM_TILE * 4;
    hipLaunchKernelGGL((ssm_bwd_kernel<T, W, VEC, true>), dim3(nblk * (p.S - 1) * p.batch), block,
                       bytes, st, p, gr);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  constexpr int bytes = ssm_bwd_lds<W, false>() * SSM_TILE * 4;
  if (hipError_t e = ensure_lds<ssm_bwd_kernel<T, W, VEC, false>>(bytes); e != hipSuccess) return e;
  hipLaunchKernelGGL((ssm_bwd_kernel<T, W, VEC, false>), dim3(nblk * p.S * p.batch), block, bytes, st,
                     p, gr);
  return hipGetLastError();
}

// 16 states at a time: the first launches leave their sums over n in memory for the last
template <typename T, bool VEC>
hipError_t bwd_waves(const Ssm& p, SsmGrad gr, hipStream_t st) {
  for (gr.n0 = 0; gr.n0 < p.N; gr.n0 += SSM_BWD_STATES) {
    const int n = p.N - gr.n0;
    gr.first = gr.n0 == 0;
    gr.last = n <= SSM_BWD_STATES;
    const hipError_t e = n <= 2   ? bwd_launch<T, 1, VEC>(p, gr, st)
                         : n <= 4 ? bwd_launch<T, 2, VEC>(p, gr, st)
                         : n <= 8 ? bwd_launch<T, 4, VEC>(p, gr, st)
                                  : bwd_launch<T, 8, VEC>(p, gr, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_ssm_bwd(const Ssm& p, const SsmGrad& gr, void* dB, void* dC, float* dA,
                          float* dD, float* dbias, bool is_bf16, bool vec, hipStream_t st) {
  hipError_t e = is_bf16 ? vec ? bwd_waves<bf16, true>(p, gr, st) : bwd_waves<bf16, false>(p, gr, st)
                 : vec   ? bwd_waves<float, true>(p, gr, st)
                         : bwd_waves<float, false>(p, gr, st);
  if (e != hipSuccess) return e;
  const int NQ = gr.NQ, parts = p.batch * p.S;
  const long long rows = (long long)p.batch * p.L;
  SumJobs jobs = {};
  for (int k = 0; k < 2; ++k) {   // dB and dC: the blocks of a group, for each group
    SumJob& j = jobs.job[jobs.n++];
    j.src = gr.part_bc + k * NQ;
    j.dst = k ? dC : dB;
    j.part_stride = rows * 2 * NQ;
    j.row_stride = 2 * NQ;
    j.out_row = (long long)p.G * p.N;
    j.out_col = 1;
    j.rows = (int)rows, j.cols = p.N, j.parts = p.gblocks, j.bf16 = is_bf16;
    j.sets = p.G, j.set_stride = p.gblocks * rows * 2 * NQ, j.out_set = p.N;
  }
  jobs.job[jobs.n++] = SumJob{gr.part_a, dA, (long long)p.N * p.E, p.E, 1, p.N, p.N, p.E, parts, 0};
  for (int k = 0; k < 2; ++k)
    if (float* dst = k ? dbias : dD)
      jobs.job[jobs.n++] =
          SumJob{gr.part_d + k * (long long)p.E, dst, 2LL * p.E, 0, 0, 1, 1, p.E, parts, 0};
  return launch_sums(jobs, st);
}

}  // namespace lz
