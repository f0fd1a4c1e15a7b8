// mxfp4.hpp -- device code shared by the kernels on microscaled 4-bit values
// (mxfp4.hip, mxfp4_gemm.hip): quantisation of a block, the activations of the
// gated linear and the store of a result.
//
// Format: 32 consecutive values of a row share one power of two, 2^(s - 127)
// with s a byte (255: the block is NaN); each value is e2m1, one of 0, 1/2, 1,
// 3/2, 2, 3, 4, 6 and their negatives. Packed rows hold two values a byte, the
// even one in the low half; a block is 16 bytes. Scales are stored by groups of
// four blocks, [ceil(K / 128)][rows][4]: the four bytes of a row and group are
// what a matrix instruction over 128 of k takes, and a tile's rows are adjacent.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace lux3d {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// s of a block from the bits of its largest magnitude, as f32: floor(log2) - 2,
// so that the largest value lies in [4, 8), and 2^-127 at least; an infinity or
// NaN (integer maxima put NaN above infinity) makes the block NaN.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top_bits) {
  const uint32_t e = top_bits >> 23;
  return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}

// Eight values, as loaded from a tensor of type T, to the four bytes of their
// codes: round to nearest even of v * 2^(127 - s), at most 6 (the convert reads
// the exponent field of its f32 scale, also where that field is 0).
template <typename T> __device__ __forceinline__ uint32_t mx_codes(const uint32_t *v, uint32_t s) {
  const float sc = __uint_as_float(s << 23);
  uint32_t r = 0;
  if constexpr (T::code == LUX3D_F32) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v[0]), __uint_as_float(v[1]), sc, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v[2]), __uint_as_float(v[3]), sc, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v[4]), __uint_as_float(v[5]), sc, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(v[6]), __uint_as_float(v[7]), sc, 3);
  } else if constexpr (T::code == LUX3D_BF16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, v[0]), sc, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, v[1]), sc, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, v[2]), sc, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, v[3]), sc, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, v[0]), sc, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, v[1]), sc, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, v[2]), sc, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2_t, v[3]), sc, 3);
  }
  return r;
}

// The largest magnitude of eight values, as f32 bits.
template <typename T> __device__ __forceinline__ uint32_t mx_top(const uint32_t *v) {
  uint32_t top = 0;
  if constexpr (T::code == LUX3D_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, v[i] & 0x7FFFFFFFu);
  } else {
    // magnitudes of 2-byte floats are ordered as their bits are
    uint32_t hi = 0, lo = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi = max(hi, v[i] & 0x7FFF0000u);
      lo = max(lo, v[i] & 0x7FFFu);
    }
    top = max(hi, lo << 16);
    if constexpr (T::code == LUX3D_F16) top = __float_as_uint(f16_bits_to_f32(top >> 16));
  }
  return top;
}

// Two codes (byte SEL of w) as T holds their values: exact in f32 and bf16, in
// f16 rounded where the block's power of two leaves its range.
template <typename T, int SEL> __device__ __forceinline__ uint32_t mx_value2(uint32_t w, float sc) {
  if constexpr (T::code == LUX3D_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, SEL));
}
// Eight codes as 2-byte values, in the layout of a matrix operand.
template <typename T> __device__ __forceinline__ u32x4_t mx_values8(uint32_t w, uint32_t s) {
  const float sc = __uint_as_float(s << 23);
  return u32x4_t{mx_value2<T, 0>(w, sc), mx_value2<T, 1>(w, sc), mx_value2<T, 2>(w, sc), mx_value2<T, 3>(w, sc)};
}

// The gated linear's activation: SiLU is v / (1 + exp(-v)), the
// tanh GELU v / (1 + exp(-2 sqrt(2 / pi) (v + 0.044715 v^3))) exactly, and the
// erf GELU v / (1 + exp(-v l(v^2))) with v l(v^2) = log(Phi(v) / Phi(-v)), l an
// even function's smooth series in v^2. So all three are v / (1 + exp2(v P(v^2)))
// with a polynomial P of their own, one code path for the three. SiLU and tanh
// GELU: 6 u for exp2, the sum, the reciprocal and the product, and the exponent's
// roundings, which are those of a v at most 4 u off (u = 2^-24): v is an f32 sum
// that is further off itself. (An exponent in two parts leaves 10 u in all and
// takes 7% of 1029 f32 rows of 1024 -> 4096.) erf: P is fitted here, degree 8
// over |v| <= 5.5, by iteratively reweighted least squares on 20,001 Chebyshev
// nodes of v^2 against log2(Phi(-v) / Phi(v)) / v: evaluated in f32 its result is
// off by 1.8e-5 of itself up to |v| = 5.5 (half a step of f16 is 4.9e-4, of bf16
// 3.9e-3); past that P stays at its last value, off by 2.4e-8. For 2-byte results;
// f32 results take mx_gelu_erf.
inline MxAct mx_act(int act) {
  switch (act) {
    case ACT_SILU: return {{-1.44269504f, 0, 0, 0, 0, 0, 0, 0, 0}, 0.f};
    case ACT_GELU_TANH: return {{-2.30220818f, -0.102943240f, 0, 0, 0, 0, 0, 0, 0}, 1e30f};
  }
  return {{-2.30221868f, -0.10480535f, 6.56670745e-05f, 0.000170996558f, -1.36602803e-05f, 6.01039289e-07f,
           -1.58674034e-08f, 2.34277681e-10f, -1.48678726e-12f},
          30.25f};
}
__device__ __forceinline__ float mx_activate(const MxAct &a, float v) {
  const float t = fminf(v * v, a.top);
  float q = a.p[8];
#pragma unroll
  for (int i = 7; i >= 0; --i) q = __builtin_fmaf(q, t, a.p[i]);
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * q));
}

// The erf GELU of f32 results: v (1 - q) or v q with q = Phi(-|v|) = erfc(z) / 2, z =
// |v| / sqrt(2), in the form of Press, Teukolsky, Vetterling & Flannery, "Numerical
// Recipes in C" (2nd ed., section 6.2): t exp(P(t) - z^2), t = 1 / (1 + z / 2), whose
// fit is off by 2 u. 12 u in all, and the exponent's roundings as above. (P of degree
// 8 over |v| <= 5.5: 300 u, most of it cancellation among its terms.)
__device__ __forceinline__ float mx_gelu_erf(float v) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(v), 0.353553391f, 1.0f));
  float p = 0.17087277f;
  p = __builtin_fmaf(p, t, -0.82215223f);
  p = __builtin_fmaf(p, t, 1.48851587f);
  p = __builtin_fmaf(p, t, -1.13520398f);
  p = __builtin_fmaf(p, t, 0.27886807f);
  p = __builtin_fmaf(p, t, -0.18628806f);
  p = __builtin_fmaf(p, t, 0.09678418f);
  p = __builtin_fmaf(p, t, 0.37409196f);
  p = __builtin_fmaf(p, t, 1.00002368f);
  p = __builtin_fmaf(p, t, -1.26551223f);
  const float w = __builtin_fmaf(__builtin_fmaf(-0.5f, v * v, p), 1.44269504f, -1.0f);
  const float q = t * __builtin_amdgcn_exp2f(w);
  return v * (v < 0 ? q : 1.0f - q);
}

// One result, rounded once to the output's type (uniform over the call).
__device__ __forceinline__ void mx_store(void *y, int dt, int64_t i, float v) {
  if (dt == LUX3D_F32) store1<F32>(y, i, v);
  else if (dt == LUX3D_BF16) store1<BF16>(y, i, v);
  else store1<F16>(y, i, v);
}

}  // namespace lux3d
