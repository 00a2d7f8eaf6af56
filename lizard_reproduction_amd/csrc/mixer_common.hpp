// What the recurrent mixers' operators share (ssm.hip, conv.hip, norm.hip): rows of
// bf16 or fp32 elements read and written through buffer resources, activations in
// fp32, and the sum of partial results in a fixed order.
#pragma once
#include "common.hpp"

namespace lz {

template <typename T>
constexpr bool IS_BF16 = sizeof(T) == 2;

// V consecutive elements of a row as loaded: packed words where the loads are vectors
// (VEC), else a word an element.  They stay packed until they are used, so that a load
// made a tile ahead holds few registers and nothing waits for it.
template <typename T, int V, bool VEC>
struct RawRow {
  static constexpr int WORDS = VEC ? (V * (int)sizeof(T) + 3) / 4 : V;
  uint32_t w[WORDS];

  __device__ __forceinline__ float at(int i) const {
    if constexpr (!IS_BF16<T>) return __builtin_bit_cast(float, w[i]);
    else if constexpr (!VEC) return __builtin_bit_cast(float, w[i] << 16);
    else return __builtin_bit_cast(float, (i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
  // rounded once, two to an instruction where they are packed
  __device__ __forceinline__ void pack(const float (&x)[V]) {
    typedef bf16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (!IS_BF16<T>)
        w[i] = __builtin_bit_cast(uint32_t, x[i]);
      else if constexpr (!VEC || V == 1)
        w[i] = __builtin_bit_cast(uint16_t, to_bf16(x[i]));
      else
        w[i] = __builtin_bit_cast(uint32_t, pair{to_bf16(x[2 * i]), to_bf16(x[2 * i + 1])});
    }
  }
};

// Elements [off, off + V) (in elements from the resource's base), zeros where !in or
// from element `left` of them on (what lies past a row's channels).
template <typename T, int V, bool VEC>
__device__ __forceinline__ RawRow<T, V, VEC> load_raw(rsrc_t r, uint32_t off, bool in, int left) {
  RawRow<T, V, VEC> o;
  constexpr int S = sizeof(T);
  if constexpr (VEC) {
    const uint32_t at = in && left > 0 ? off * S : OOB;
    constexpr int B = V * S;
    if constexpr (B == 2) {
      o.w[0] = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
    } else if constexpr (B == 4) {
      o.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    } else if constexpr (B == 8) {
      const auto v = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0));
      o.w[0] = v.x, o.w[1] = v.y;
    } else {
#pragma unroll
      for (int k = 0; k < B / 16; ++k) {
        const uint4 v = bload16(r, at + 16 * k);
        o.w[4 * k] = v.x, o.w[4 * k + 1] = v.y, o.w[4 * k + 2] = v.z, o.w[4 * k + 3] = v.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t at = in && i < left ? (off + i) * S : OOB;
      if constexpr (S == 2) o.w[i] = __builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
      else o.w[i] = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0);
    }
  }
  return o;
}

template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_raw(rsrc_t r, uint32_t off, bool in, int left,
                                          const RawRow<T, V, VEC>& o) {
  constexpr int S = sizeof(T);
  if constexpr (VEC) {
    const uint32_t at = in && left > 0 ? off * S : OOB;
    constexpr int B = V * S;
    if constexpr (B == 2) {
      __builtin_amdgcn_raw_buffer_store_b16((uint16_t)o.w[0], r, at, 0, 0);
    } else if constexpr (B == 4) {
      __builtin_amdgcn_raw_buffer_store_b32(o.w[0], r, at, 0, 0);
    } else if constexpr (B == 8) {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      __builtin_amdgcn_raw_buffer_store_b64(u32x2{o.w[0], o.w[1]}, r, at, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < B / 16; ++k)
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4{o.w[4 * k], o.w[4 * k + 1], o.w[4 * k + 2], o.w[4 * k + 3]}, r, at + 16 * k, 0, 0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t at = in && i < left ? (off + i) * S : OOB;
      if constexpr (S == 2) __builtin_amdgcn_raw_buffer_store_b16((uint16_t)o.w[i], r, at, 0, 0);
      else __builtin_amdgcn_raw_buffer_store_b32(o.w[i], r, at, 0, 0);
    }
  }
}

// N channels of a row through a pointer of the lane's own, as vectors of up to 16 bytes at
// any alignment (VEC), else element by element, `left` of them.  Rows are clamped into the
// tensor by the callers and what does not exist is selected away after the load, so no
// branch holds loads apart.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

template <typename T, bool VEC, int N>
struct Cols {
  RawRow<T, N, VEC> r;
  static constexpr int BYTES = N * (int)sizeof(T);
  __device__ __forceinline__ void load(const T* p, int left) {
    if constexpr (VEC && BYTES == 8) {
      const u32x2_any v = *reinterpret_cast<const u32x2_any*>(p);
      r.w[0] = v[0], r.w[1] = v[1];
    } else if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < BYTES / 16; ++k) {
        const u32x4_any v = reinterpret_cast<const u32x4_any*>(p)[k];
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[4 * k + i] = v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const T v = p[i < left ? i : 0];
        if constexpr (IS_BF16<T>) r.w[i] = __builtin_bit_cast(uint16_t, v);
        else r.w[i] = __builtin_bit_cast(uint32_t, v);
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int left) const {
    if constexpr (VEC && BYTES == 8) {
      *reinterpret_cast<u32x2_any*>(p) = u32x2_any{r.w[0], r.w[1]};
    } else if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < BYTES / 16; ++k)
        reinterpret_cast<u32x4_any*>(p)[k] =
            u32x4_any{r.w[4 * k], r.w[4 * k + 1], r.w[4 * k + 2], r.w[4 * k + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < left) p[i] = (T)r.at(i);
    }
  }
};

// A resource from base on that takes every offset under 2 GiB: the loads and stores here
// pass OOB for what a row or a tile does not have.  Callers rebase it every few rows, in
// 64 bits, so the 32-bit offsets within never pass a tile.
template <typename T>
__device__ __forceinline__ rsrc_t open_rsrc(const T* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), (short)0, 0x7fffffff, RSRC_WORD3);
}

__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + fexp(-x));   // e^-x past fp32: 1 / inf = 0
}

// log(1 + e^x) = max(x, 0) + log(1 + e) with e = e^-|x| in [0, 1], and its slope 1 / (1 +
// e^-x).  log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3: s times a polynomial of degree
// 4 in s^2, which interpolates 2 atanh(s) / s at the Chebyshev nodes of [0, 1/9], within 4e-9
// of it; four units in the last place in all.  (The hardware's log of 1 + e would lose e's
// low bits, and small steps are what a trained dt gives.)
__device__ __forceinline__ float softplus_of(float x, float e) {
  const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
  float p = 0.28157780f;
  p = fmaf(p, q, 0.27965158f);
  p = fmaf(p, q, 0.40024596f);
  p = fmaf(p, q, 0.66666320f);
  p = fmaf(p, q, 2.f);
  return fmaf(s, p, fmaxf(x, 0.f));
}

__device__ __forceinline__ float softplus(float x) { return softplus_of(x, fexp(-fabsf(x))); }

__device__ __forceinline__ float softplus_slope(float x, float& slope) {
  const float e = fexp(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + e);
  slope = x >= 0.f ? r : e * r;
  return softplus_of(x, e);
}

// x of another lane of this lane's row of 16, or of its quad, as an operand of the
// instruction that uses it (DPP).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xb1, DPP_XOR2 = 0x4e;          // quad_perm [1,0,3,2], [2,3,0,1]
constexpr int DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;   // lane 7 - i of its 8, 15 - i of its 16
constexpr int DPP_ROR8 = 0x128;                          // lane i + 8 mod 16
constexpr int DPP_BCAST = 0x150;                         // + k: lane k of the row, to all of it

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

// The sums over each `lanes` (a power of two, uniform) consecutive lanes, in all of them.
// (The empty asm has the comparisons made where they are: kept from before a loop, they come
// out of vector registers.)
template <int N>
__device__ __forceinline__ void lanes_sum(float (&v)[N], int lanes) {
  asm volatile("" : "+s"(lanes));
  auto add = [&](auto other) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = other(v[i]);
  };
  auto quads = [&] {
    add([](float x) { return x + dpp<DPP_XOR1>(x); });
    add([](float x) { return x + dpp<DPP_XOR2>(x); });
  };
  if (lanes >= 16) {
    quads();
    add([](float x) { return x + dpp<DPP_HALF_MIRROR>(x); });
    add([](float x) { return x + dpp<DPP_MIRROR>(x); });
    if (lanes >= 32) add([](float x) { return swap_add<true>(x, x); });
    if (lanes >= 64) add([](float x) { return swap_add<false>(x, x); });
  } else if (lanes >= 4) {
    quads();
    if (lanes >= 8) add([](float x) { return x + dpp<DPP_HALF_MIRROR>(x); });
  } else if (lanes >= 2) {
    add([](float x) { return x + dpp<DPP_XOR1>(x); });
  }
}

// Sums of partial results in the order of their index, by one launch.  A job sums, for
// each of `sets` x `rows` x `cols` outputs, `parts` values `part_stride` floats apart that
// begin at src + set * set_stride + row * row_stride + col; output (set, row, col) goes to
// dst + set * out_set + row * out_row + col * out_col, as bf16 or float.
struct SumJob {
  const float* src;
  void* dst;
  long long part_stride, row_stride, out_row, out_col;
  int rows, cols, parts, bf16;
  int sets = 1;
  long long set_stride = 0, out_set = 0;
};
constexpr int SUM_JOBS = 6;
struct SumJobs {
  SumJob job[SUM_JOBS];
  int n;
};
hipError_t launch_sums(const SumJobs& jobs, hipStream_t st);

}  // namespace lz
