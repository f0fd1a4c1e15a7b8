// attn_tiles.hpp -- device helpers of the attention kernels (attention.hip,
// prefix_attention.hip): matrix-core operations of the 2-byte types, the LDS
// swizzles of K and V rows, lane exchanges and the workgroup order.
#pragma once

#include "common.hpp"

namespace lux3d {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Mma;
template <> struct Mma<BF16> {
  typedef bf16x8_t op_t;
  __device__ __forceinline__ static f32x16_t run(op_t a, op_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  __device__ __forceinline__ static float sum2(uint32_t pair, float acc) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t one = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), one, acc, false);
  }
};
template <> struct Mma<F16> {
  typedef f16x8_t op_t;
  __device__ __forceinline__ static f32x16_t run(op_t a, op_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  __device__ __forceinline__ static float sum2(uint32_t pair, float acc) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f16x2_t one = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pair), one, acc, false);
  }
};

// the same into element e of three packed operand vectors
__device__ __forceinline__ void split3_into(float a, float b, u32x4_t &x1, u32x4_t &x2, u32x4_t &x3, int e) {
  const Split3 r = split3_bf16(a, b);
  x1[e] = r.t1;
  x2[e] = r.t2;
  x3[e] = r.t3;
}

// Slots of the 16-byte chunks of K / V rows of D 2-byte elements in LDS
// without padding: chunk c of row r in slot c ^ k_swz(r) (v_swz(r)). A K
// fragment read takes one chunk of 16 consecutive rows at a time, a V^T read
// four consecutive chunks of four rows; each such 256 bytes then cover all 64
// banks once. (With one swizzle c ^ ((r & 7) * D / 64) for both, every read
// conflicted two ways: half of the LDS cycles.)
template <int D> __device__ __forceinline__ int k_swz(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
template <int D> __device__ __forceinline__ int v_swz(int r) { return D == 128 ? (r & 3) << 2 : (r & 2) << 1; }

// Counts as a use of x at this place.
__device__ __forceinline__ void keep(const f32x16_t &x) { asm volatile("" ::"v"(x)); }

// The value the partner lane (lane ^ 32) holds, paired with this lane's own:
// v_permlane32_swap exchanges the two 32-lane halves.
__device__ __forceinline__ float half_swap_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Logical workgroup id for physical id `pid` of `n`: XCD x (pid % 8) gets the
// contiguous logical range [start_x, start_x + count_x).
__device__ __forceinline__ int64_t xcd_logical_id(int64_t pid, int64_t n) {
  const int64_t per = n / 8, rem = n % 8, xcd = pid % 8, idx = pid / 8;
  return (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + idx;
}

}  // namespace lux3d
