// Arguments of the selective state space scan's kernels (ssm.hip, ssm_bwd.hip) and the
// walk over a tile that both directions begin with.
#pragma once
#include <type_traits>
#include <utility>

#include "mixer_common.hpp"

namespace lz {

// Layout of the work.  A workgroup takes 64 channels of one group and one sequence (or a
// segment of it) and walks it in tiles of 16 tokens.  In its W scan waves a lane is a
// channel; a wave holds NS states in registers, two or four (and another NS from NS (w + W)
// on with NP = 2) in the forward, two in the backward.  Helper waves turn the next tile's
// rows into delta, u and the like while the scan waves walk this one, and the last tile's
// sums into rows: one barrier a tile, and other waves to switch to while one waits.  (With
// the scan waves doing both, two barriers a tile, the training pass of 8192 tokens x 4096
// channels x 16 states took 857 us where this took 738.)
// In LDS a tile is rows of the 64 channels: a thread's share of a row is one vector, a
// wave's read of a token 64 consecutive floats (channels of 16 tokens each, 20 floats
// apart, made the transposed writes and reads conflict: 40 % of the forward's time).
constexpr int SSM_CH = 64, SSM_TT = 16, SSM_MAX_STATE = 64;
constexpr int SSM_TILE = SSM_CH * SSM_TT;

struct Ssm {
  const void *x, *dt, *z, *B, *C;
  const float *A, *D, *bias;
  const float* state_in;
  float* state_out;
  const int* lengths;
  void* y;
  float* mixed;    // [B, L, E]: sum_n C h + D x, where z gates it, for the backward
  float* saved;    // [B, tiles, N, E]: the state before each tile, likewise
  float* rec;      // [B, S - 1, N, E]: a segment's own state, from zero
  float* dsum;     // [B, S - 1, E]: its sum of delta
  long long x_b, dt_b, z_b, B_b, C_b, y_b;   // elements from one sequence to the next
  int x_t, dt_t, z_t, B_t, C_t;              // from one token to the next
  int B_g, C_g;                              // from one group to the next
  int batch, L, E, N, G, Eg, gblocks;        // gblocks: 64-channel blocks of a group
  int tiles, seg_tiles, S, softplus;
};

// Gradients (ssm_bwd.hip)
struct SsmGrad {
  const void* dy;
  void *dx, *ddt, *dz;   // [B, L, E]
  float* part_bc;        // [blocks, B, L, 2, NQ]: a block's share of dB and dC
  float* part_a;         // [B S, N, E]
  float* part_d;         // [B S, 2, E]: of dD and ddt_bias
  float* rec;            // as Ssm's, of the reverse walk
  float* dsum;
  float* acc;            // [2][B, L, E]: sums over the states of earlier launches
  long long acc_step;    // B L E
  int n0, first, last;   // this launch's first state; whether it is the first, the last
  int NQ;                // padded states in part_bc
};

// Helper waves of the backward (the forward's are chosen with its scan waves): its registers
// leave room for twelve waves.  A thread of theirs takes a vector of V channels of one row of
// a tile.
constexpr int SSM_HELPERS = 4, SSM_V = SSM_TILE / (64 * SSM_HELPERS);
constexpr int SSM_COLS = SSM_CH / SSM_V, SSM_ROWS = 64 * SSM_HELPERS / SSM_COLS;
static_assert(SSM_V == 4 && SSM_ROWS == SSM_TT, "a thread, a vector of the tile");

template <class F, int... K>
__device__ __forceinline__ void static_for_impl(F f, std::integer_sequence<int, K...>) {
  (f(std::integral_constant<int, K>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// A thread's vector of a tile
template <int V>
__device__ __forceinline__ void put_row(float* to, const float (&v)[V]) {
  typedef float vec __attribute__((ext_vector_type(V)));
  vec x;
#pragma unroll
  for (int k = 0; k < V; ++k) x[k] = v[k];
  *reinterpret_cast<vec*>(to) = x;
}
template <int V>
__device__ __forceinline__ void add_row(float (&v)[V], const float* from) {
  typedef float vec __attribute__((ext_vector_type(V)));
  const vec x = *reinterpret_cast<const vec*>(from);
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] += x[k];
}
// Four tokens of a lane's channel
__device__ __forceinline__ f32x4 get_tokens(const float* tile, int t, int lane) {
  const float* p = tile + t * SSM_CH + lane;
  return f32x4{p[0], p[SSM_CH], p[2 * SSM_CH], p[3 * SSM_CH]};
}
__device__ __forceinline__ void put_tokens(float* tile, int t, int lane, const f32x4& v) {
  float* p = tile + t * SSM_CH + lane;
#pragma unroll
  for (int k = 0; k < 4; ++k) p[k * SSM_CH] = v[k];
}

// B or C of a tile for a wave's NS states (2 or 4): register i of a lane holds token
// (16 / NS) i + (lane % 16) / NS, state lane % NS, so that the k-th token's state n of
// register i is lane NS k + n of every row of 16, which a DPP operand broadcasts.
template <typename T, int NS>
struct SsmVec {
  static constexpr int TOKENS = 16 / NS;   // a register
  std::conditional_t<IS_BF16<T>, uint16_t, uint32_t> w[NS];   // as loaded until they are used
  __device__ __forceinline__ void load(const T* base, int rows, int pitch, int N, int n0, int lane) {
    const rsrc_t r = open_rsrc(base);
    const int n = n0 + lane % NS;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int t = TOKENS * i + lane % 16 / NS;
      const uint32_t at = t < rows && n < N ? (uint32_t)(t * pitch + n) * (uint32_t)sizeof(T) : OOB;
      if constexpr (IS_BF16<T>) w[i] = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
      else w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    }
  }
  __device__ __forceinline__ float at(int i) const {
    return __builtin_bit_cast(float, IS_BF16<T> ? (uint32_t)w[i] << 16 : (uint32_t)w[i]);
  }
};

// y[t] = sum_n v(K + NS t + n) h[t][n] (ADD: added to y[t]) for four tokens t, v(k) lane k of
// a row of 16: the compiler folds the broadcast into a product but not into a multiply-add,
// so these are written out, behind the two wait states that a DPP operand asks for after its
// register was written.
#define LZ_DPP(op, t, k, n) \
  op " %" #t ", %4, %" #n " row_newbcast:%" #k " row_mask:0xf bank_mask:0xf\n"
#define LZ_FIRST LZ_DPP("v_mul_f32_dpp", 0, 13, 5) LZ_DPP("v_mul_f32_dpp", 1, 15, 7) \
  LZ_DPP("v_mul_f32_dpp", 2, 17, 9) LZ_DPP("v_mul_f32_dpp", 3, 19, 11)
#define LZ_DOT(t, k, n) LZ_DPP("v_fmac_f32_dpp", t, k, n)
#define LZ_FIRST_ADD LZ_DOT(0, 13, 5) LZ_DOT(1, 15, 7) LZ_DOT(2, 17, 9) LZ_DOT(3, 19, 11)
#define LZ_REST LZ_DOT(0, 14, 6) LZ_DOT(1, 16, 8) LZ_DOT(2, 18, 10) LZ_DOT(3, 20, 12)
#define LZ_INS                                                                                 \
  "v"(v), "v"(h[0][0]), "v"(h[0][1]), "v"(h[1][0]), "v"(h[1][1]), "v"(h[2][0]), "v"(h[2][1]), \
      "v"(h[3][0]), "v"(h[3][1]), "n"(K), "n"(K + 1), "n"(K + 2), "n"(K + 3), "n"(K + 4),     \
      "n"(K + 5), "n"(K + 6), "n"(K + 7)
template <int K, bool ADD>
__device__ __forceinline__ void ssm_dots(f32x4& y, float v, const float (&h)[4][2]) {
  float y0, y1, y2, y3;
  if constexpr (ADD) {
    y0 = y[0], y1 = y[1], y2 = y[2], y3 = y[3];
    asm("s_nop 1\n" LZ_FIRST_ADD LZ_REST : "+&v"(y0), "+&v"(y1), "+&v"(y2), "+&v"(y3) : LZ_INS);
  } else {
    asm("s_nop 1\n" LZ_FIRST LZ_REST : "=&v"(y0), "=&v"(y1), "=&v"(y2), "=&v"(y3) : LZ_INS);
  }
  y = f32x4{y0, y1, y2, y3};
}
#undef LZ_FIRST
#undef LZ_FIRST_ADD
#undef LZ_REST
#undef LZ_INS
#undef LZ_DOT
#undef LZ_DPP
#define LZ_DPP(op, t, k, n) \
  op " %" #t ", %4, %" #n " row_newbcast:" #k " row_mask:0xf bank_mask:0xf\n"
#define LZ_FIRST LZ_DPP("v_mul_f32_dpp", 0, 0, 5) LZ_DPP("v_mul_f32_dpp", 1, 4, 9) \
  LZ_DPP("v_mul_f32_dpp", 2, 8, 13) LZ_DPP("v_mul_f32_dpp", 3, 12, 17)
#define LZ_DOT(t, k, n) LZ_DPP("v_fmac_f32_dpp", t, k, n)
#define LZ_FIRST_ADD LZ_DOT(0, 0, 5) LZ_DOT(1, 4, 9) LZ_DOT(2, 8, 13) LZ_DOT(3, 12, 17)
#define LZ_REST                                                     \
  LZ_DOT(0, 1, 6) LZ_DOT(1, 5, 10) LZ_DOT(2, 9, 14) LZ_DOT(3, 13, 18)  \
  LZ_DOT(0, 2, 7) LZ_DOT(1, 6, 11) LZ_DOT(2, 10, 15) LZ_DOT(3, 14, 19) \
  LZ_DOT(0, 3, 8) LZ_DOT(1, 7, 12) LZ_DOT(2, 11, 16) LZ_DOT(3, 15, 20)
#define LZ_INS                                                                                 \
  "v"(v), "v"(h[0][0]), "v"(h[0][1]), "v"(h[0][2]), "v"(h[0][3]), "v"(h[1][0]), "v"(h[1][1]), \
      "v"(h[1][2]), "v"(h[1][3]), "v"(h[2][0]), "v"(h[2][1]), "v"(h[2][2]), "v"(h[2][3]),     \
      "v"(h[3][0]), "v"(h[3][1]), "v"(h[3][2]), "v"(h[3][3])
template <int, bool ADD>
__device__ __forceinline__ void ssm_dots(f32x4& y, float v, const float (&h)[4][4]) {
  float y0, y1, y2, y3;
  if constexpr (ADD) {
    y0 = y[0], y1 = y[1], y2 = y[2], y3 = y[3];
    asm("s_nop 1\n" LZ_FIRST_ADD LZ_REST : "+&v"(y0), "+&v"(y1), "+&v"(y2), "+&v"(y3) : LZ_INS);
  } else {
    asm("s_nop 1\n" LZ_FIRST LZ_REST : "=&v"(y0), "=&v"(y1), "=&v"(y2), "=&v"(y3) : LZ_INS);
  }
  y = f32x4{y0, y1, y2, y3};
}
#undef LZ_FIRST
#undef LZ_FIRST_ADD
#undef LZ_REST
#undef LZ_INS
#undef LZ_DOT
#undef LZ_DPP

// c[n] + v(K + n) x, likewise
template <int K>
__device__ __forceinline__ void ssm_fma2(float (&g)[2], float v, float x, const float (&c)[2]) {
  float g0 = c[0], g1 = c[1];
  asm("s_nop 1\n"
      "v_fmac_f32_dpp %0, %2, %3 row_newbcast:%4 row_mask:0xf bank_mask:0xf\n"
      "v_fmac_f32_dpp %1, %2, %3 row_newbcast:%5 row_mask:0xf bank_mask:0xf\n"
      : "+&v"(g0), "+&v"(g1)
      : "v"(v), "v"(x), "n"(K), "n"(K + 1));
  g[0] = g0, g[1] = g1;
}

// Where a workgroup works
struct SsmPlace {
  int b, s, blk, g, c0, cols;   // sequence, segment, block; group, first channel, channels
  int len, tile0, tile1;        // the sequence's length, the segment's tiles
  __device__ __forceinline__ SsmPlace(const Ssm& p, int segments) {
    const int nblk = p.G * p.gblocks;
    int i = blockIdx.x;
    blk = i % nblk;
    i /= nblk;
    s = i % segments;
    b = i / segments;
    g = blk / p.gblocks;
    const int first = (blk - g * p.gblocks) * SSM_CH;
    c0 = g * p.Eg + first;
    cols = min(SSM_CH, p.Eg - first);
    len = p.lengths ? max(0, min(p.L, p.lengths[b])) : p.L;
    tile0 = s * p.seg_tiles;
    tile1 = min(p.tiles, tile0 + p.seg_tiles);
  }
};

// States the backward takes a launch, and N padded to whole launches
constexpr int SSM_BWD_STATES = 16;
inline int ssm_bwd_padded(int N) {
  return N <= 2 ? 2 : N <= 4 ? 4 : N <= 8 ? 8 : (N + 15) / 16 * 16;
}

int ssm_segments(int batch, int G, int Eg, int L, bool backward);
hipError_t launch_ssm_fwd(const Ssm& p, bool is_bf16, bool vec, hipStream_t st);
hipError_t launch_ssm_step(const Ssm& p, float* state, bool is_bf16, hipStream_t st);
hipError_t launch_ssm_bwd(const Ssm& p, const SsmGrad& g, void* dB, void* dC, float* dA,
                          float* dD, float* dbias, bool is_bf16, bool vec, hipStream_t st);

}  // namespace lz
