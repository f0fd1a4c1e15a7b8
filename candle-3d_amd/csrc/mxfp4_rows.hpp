// mxfp4_rows.hpp -- few rows of a linear layer on microscaled 4-bit weights: a
// workgroup's share, for the kernel of few rows (mxfp4.hip) and for the rows past
// the last tile of the kernel of many (mxfp4_gemm.hip).
#pragma once

#include <type_traits>

#include "mxfp4.hpp"

namespace lux3d {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

// A workgroup owns NT tiles of 16 weight rows (of each matrix) and MT tiles of
// 16 rows of x; its NW wavefronts take groups of 128 of k in turn and add their
// sums in wavefront order through LDS. Lane l holds row l % 16 and block l / 16 of
// the group of either operand: 16 bytes of a packed row, 32 values of a plain one.
//   fp4    one v_mfma_scale_f32_16x16x128_f8f6f4 a group, each lane's scale its
//          own block's; plain x is quantised in the lane that holds the block
//   plain  four v_mfma_f32_16x16x32 on the block's four eighths; the weights'
//          values are exact in bf16; f32 x in three exact bf16 terms
// Bound by latency where the weights are a few MB (1 row of 2048 -> 8192, bf16: 4.2
// us, an empty launch 2.2), by their bytes where they are many (4096 -> 32000: 15.7
// us, 4.4 TB/s), and by x's loads and conversions with every row more (16: 22).
// Rows m0 to M - 1 at most, outputs from n0 on. lds: mx_rows_lds bytes.
template <bool GATED, int MT, int NT, int NW> constexpr int mx_rows_lds = NW * (GATED ? 2 : 1) * NT * MT * 1024;

template <typename X, bool FP4, bool GATED, int MT, int NT, int NW>
__device__ __forceinline__ void mx_rows_tile(const MxLinearParams &p, const MxAct &act, int64_t m0, int64_t M, int64_t n0, float *lds) {
  constexpr bool PACKED = std::is_void_v<X>;
  constexpr int NM = GATED ? 2 * NT : NT;  // weight tiles: the gate's behind the others
  float(*const part)[NM][MT][256] = reinterpret_cast<float(*)[NM][MT][256]>(lds);
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4, l16 = lane & 15;
  const int64_t nb = p.K / 32, groups = (nb + 3) / 4;
  f32x4_t acc[NM][MT];
#pragma unroll
  for (int j = 0; j < NM; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = f32x4_t{};
  // what a lane holds of a group: its block of each matrix and of each row tile
  constexpr int XN = PACKED ? 1 : 2 * std::conditional_t<PACKED, F32, X>::bytes;  // 16-byte pieces of x's block
  struct Group {
    uint4 w[NM], x[MT][XN];
    uint32_t sw[NM], sx[MT];
  };
  auto load = [&](Group &q, int64_t c) {
    const int64_t b = 4 * c + g;
    const bool live = b < nb;  // a last group may have fewer than four blocks: the others count as 0
#pragma unroll
    for (int j = 0; j < NM; ++j) {
      const int64_t at = n0 + 16 * (j % NT) + l16, n = at < p.N ? at : p.N - 1;  // past N: clamped, never stored
      q.w[j] = ld16<false>(p.w[j / NT] + n * (p.K / 2) + (live ? b : nb - 1) * 16);
      q.sw[j] = live ? p.ws[j / NT][(c * p.N + n) * 4 + g] : 0;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + 16 * i + l16;
#pragma unroll
      for (int e = 0; e < XN; ++e) q.x[i][e] = make_uint4(0, 0, 0, 0);
      q.sx[i] = 0;
      if (live && m < M) {
        if constexpr (PACKED) {
          q.x[i][0] = ld16<false>(p.xq + m * (p.K / 2) + b * 16);
          q.sx[i] = p.xs[(c * p.xs_rows + m) * 4 + g];
        } else {
          const char *src = reinterpret_cast<const char *>(p.x) + (m * p.ldx + b * 32) * X::bytes;
#pragma unroll
          for (int e = 0; e < XN; ++e) q.x[i][e] = ld16<false>(src + 16 * e);
        }
      }
    }
  };
  auto products = [&](Group &q) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (FP4) {
        u32x4_t xc;
        uint32_t sx = q.sx[i];
        if constexpr (PACKED) {
          xc = u32x4_t{q.x[i][0].x, q.x[i][0].y, q.x[i][0].z, q.x[i][0].w};
        } else {
          uint32_t v[4 * XN];
#pragma unroll
          for (int e = 0; e < XN; ++e) {
            v[4 * e] = q.x[i][e].x;
            v[4 * e + 1] = q.x[i][e].y;
            v[4 * e + 2] = q.x[i][e].z;
            v[4 * e + 3] = q.x[i][e].w;
          }
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, mx_top<X>(v + e * XN));
          sx = mx_scale(top);
#pragma unroll
          for (int e = 0; e < 4; ++e) xc[e] = mx_codes<X>(v + e * XN, sx);
        }
        const i32x8_t xb = {(int)xc[0], (int)xc[1], (int)xc[2], (int)xc[3], 0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NM; ++j) {
          const i32x8_t wa = {(int)q.w[j].x, (int)q.w[j].y, (int)q.w[j].z, (int)q.w[j].w, 0, 0, 0, 0};
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc[j][i], 4, 4, 0, (int)q.sw[j], 0, (int)sx);
        }
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          u32x4_t x1, x2, x3;
          if constexpr (X::code == LUX3D_F32) {
            const uint4 a = q.x[i][2 * s], c = q.x[i][2 * s + 1];
            const uint32_t f[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const Split3 r = split3_bf16(__uint_as_float(f[2 * e]), __uint_as_float(f[2 * e + 1]));
              x1[e] = r.t1;
              x2[e] = r.t2;
              x3[e] = r.t3;
            }
          } else {
            x1 = u32x4_t{q.x[i][s].x, q.x[i][s].y, q.x[i][s].z, q.x[i][s].w};
          }
#pragma unroll
          for (int j = 0; j < NM; ++j) {
            const uint32_t ws = s == 0 ? q.w[j].x : s == 1 ? q.w[j].y : s == 2 ? q.w[j].z : q.w[j].w;
            if constexpr (X::code == LUX3D_F16) {
              acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, mx_values8<F16>(ws, q.sw[j])),
                                                                 __builtin_bit_cast(f16x8_t, x1), acc[j][i], 0, 0, 0);
            } else {
              const bf16x8_t wv = __builtin_bit_cast(bf16x8_t, mx_values8<BF16>(ws, q.sw[j]));
              if constexpr (X::code == LUX3D_F32) {
                acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, __builtin_bit_cast(bf16x8_t, x3), acc[j][i], 0, 0, 0);
                acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, __builtin_bit_cast(bf16x8_t, x2), acc[j][i], 0, 0, 0);
              }
              acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, __builtin_bit_cast(bf16x8_t, x1), acc[j][i], 0, 0, 0);
            }
          }
        }
      }
    }
  };
  for (int64_t c = wave; c < groups; c += NW) {
    Group q;
    load(q, c);
    products(q);
  }
  // lane holds weight rows 4 g + e, x row l16 of each tile
#pragma unroll
  for (int j = 0; j < NM; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][j][i][e * 64 + lane] = acc[j][i][e];
  __syncthreads();
  for (int o = t; o < MT * NT * 256; o += 64 * NW) {
    const int c16 = o % (16 * NT), tile = c16 >> 4, c = c16 & 15, r = o / (16 * NT) & 15, i = o / (256 * NT);
    const int at = (c & 3) * 64 + (c >> 2) * 16 + r;
    const int64_t row = m0 + 16 * i + r, col = n0 + c16;
    if (row >= M || col >= p.N) continue;
    float v[2];
#pragma unroll
    for (int j = 0; j < NM / NT; ++j) {
      v[j] = part[0][j * NT + tile][i][at];
#pragma unroll
      for (int k = 1; k < NW; ++k) v[j] += part[k][j * NT + tile][i][at];
      if (p.bias[j]) v[j] += p.bias[j][col];
    }
    float y = v[0];
    if constexpr (GATED) y *= p.y_dt == LUX3D_F32 && p.act == ACT_GELU_ERF ? mx_gelu_erf(v[1]) : mx_activate(act, v[1]);
    mx_store(p.y, p.y_dt, row * p.ldy + col, y);
  }
}

}  // namespace lux3d
