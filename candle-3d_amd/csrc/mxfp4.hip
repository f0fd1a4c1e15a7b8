// mxfp4.hip -- microscaled 4-bit values on gfx950: quantisation, its inverse,
// and the linear layers of few rows (mxfp4.hpp: the format).
#include <type_traits>

#include "mxfp4.hpp"

namespace lux3d {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

// ---- quantisation ---------------------------------------------------------------
//
// A stream: x read once, 17 / 32 byte a value written. A workgroup takes 4 R rows
// x 512 values; a wavefront reads a row's 512 with 8 values a lane (4 lanes a
// block, the block's maximum by two DPP steps), R rows in flight, and writes 256
// contiguous bytes of codes a row. The scales go through LDS: a group's bytes of
// 4 R rows are adjacent. R is 4, and 2 where that leaves fewer than two workgroups
// a CU (us with R of 8 / 4 / 2: 777 x 1120 bf16 3.4 / 2.8 / 2.5, 1029 x 1024 f32
// 4.8 / 3.0 / 2.6, 4098 x 2048 bf16 5.8 / 5.0 / 5.0, 9001 x 1536 8.2 / 7.4 / 7.9,
// 64000 x 1536 41.1 / 40.4 / 43.9, 8192 x 2048 f32 17.0 / 14.8 / 14.7: 5.1 to 6.2
// TB/s where the launch does not count).
constexpr int kQuantCols = 512;
inline int64_t mx_quant_tiles(int64_t rows, int64_t k, int r) { return (k + kQuantCols - 1) / kQuantCols * ((rows + 4 * r - 1) / (4 * r)); }

template <typename T, int R>
__global__ __launch_bounds__(256) void mx_quantize_kernel(MxQuantParams p) {
  constexpr int NV = T::bytes == 4 ? 2 : 1;  // 16-byte loads a lane and row
  __shared__ uint32_t sc[4][4 * R];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t tk = (p.K + kQuantCols - 1) / kQuantCols, rt = (int64_t)blockIdx.x / tk, kt = blockIdx.x - rt * tk;
  const int64_t r0 = rt * (4 * R), k = kt * kQuantCols + lane * 8;
  const bool live = k < p.K;
  uint32_t v[R][4 * NV];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t r = r0 + wave * R + i;
#pragma unroll
    for (int j = 0; j < 4 * NV; ++j) v[i][j] = 0;
    if (live && r < p.M) {
      const char *src = reinterpret_cast<const char *>(p.x) + (r * p.ldx + k) * T::bytes;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint4 u = ld16(src + 16 * j);
        v[i][4 * j] = u.x;
        v[i][4 * j + 1] = u.y;
        v[i][4 * j + 2] = u.z;
        v[i][4 * j + 3] = u.w;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t r = r0 + wave * R + i;
    uint32_t top = mx_top<T>(v[i]);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, DPP_XOR1, 0xF, 0xF, false));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, DPP_XOR2, 0xF, 0xF, false));
    const uint32_t s = mx_scale(top);  // values past K count as 0: so do the scales that fill up the last group
    const uint32_t codes = mx_codes<T>(v[i], s);
    if (live && r < p.M) *reinterpret_cast<uint32_t *>(p.q + (r * p.K + k) / 2) = codes;
    if ((lane & 3) == 0) reinterpret_cast<uint8_t *>(&sc[lane >> 4][wave * R + i])[(lane >> 2) & 3] = (uint8_t)s;
  }
  __syncthreads();
  const int64_t g = kt * 4 + t / (4 * R), r = r0 + t % (4 * R);
  if (t < 16 * R && g * 128 < p.K && r < p.M) reinterpret_cast<uint32_t *>(p.s)[g * p.M + r] = sc[t / (4 * R)][t % (4 * R)];
}

// ---- and back -------------------------------------------------------------------
//
// The same tiles, R rows of a wavefront in flight. A lane writes 16 bytes and the
// next lane the 16 behind them: 8 values of a 2-byte type, 4 of f32, which takes
// the row's half in two steps (16 values a lane and four stores 64 bytes apart
// instead: 8192 x 2048 f32 50 us against 12).
template <typename T, int R>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxDequantParams p) {
  constexpr int V = 16 / T::bytes, STEPS = 8 / V;  // values a lane and step
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t tk = (p.K + kQuantCols - 1) / kQuantCols, rt = (int64_t)blockIdx.x / tk, kt = blockIdx.x - rt * tk;
  const int64_t r0 = rt * (4 * R) + wave * R;
#pragma unroll
  for (int step = 0; step < STEPS; ++step) {
    const int64_t k = kt * kQuantCols + step * (kQuantCols / STEPS) + lane * V;
    if (k >= p.K) return;
    uint32_t c[R], s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i < p.M ? r0 + i : p.M - 1;
      const uint8_t *src = p.q + (r * p.K + k) / 2;
      if constexpr (V == 8) c[i] = *reinterpret_cast<const uint32_t *>(src);
      else c[i] = *reinterpret_cast<const uint16_t *>(src);
      s[i] = p.s[((k >> 7) * p.M + r) * 4 + ((k >> 5) & 3)];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (r0 + i >= p.M) break;
      void *dst = reinterpret_cast<char *>(p.y) + ((r0 + i) * p.ldy + k) * T::bytes;
      if constexpr (V == 8) {
        const u32x4_t v = mx_values8<T>(c[i], s[i]);
        st16(dst, make_uint4(v[0], v[1], v[2], v[3]));
      } else {
        const float sc = __uint_as_float(s[i] << 23);
        const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], sc, 1);
        st16(dst, make_uint4(__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])));
      }
    }
  }
}

// ---- linear, few rows -----------------------------------------------------------
//
// A workgroup owns NT tiles of 16 weight rows (of each matrix) and MT tiles of
// 16 rows of x; its NW wavefronts take groups of 128 of k in turn and add their sums in
// wavefront order through LDS. Lane l holds row l % 16 and block l / 16 of the
// group of either operand: 16 bytes of a packed row, 32 values of a plain one.
//   fp4    one v_mfma_scale_f32_16x16x128_f8f6f4 a group, each lane's scale its
//          own block's; plain x is quantised in the lane that holds the block
//   plain  four v_mfma_f32_16x16x32 on the block's four eighths; the weights'
//          values are exact in bf16; f32 x in three exact bf16 terms
template <typename X, bool FP4, bool GATED, int MT, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void mx_rows_kernel(MxLinearParams p, MxAct act) {
  constexpr bool PACKED = std::is_void_v<X>;
  constexpr int NM = GATED ? 2 * NT : NT;  // weight tiles: the gate's behind the others
  __shared__ float part[NW][NM][MT][256];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4, l16 = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NT, m0 = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 16 * MT;
  if (m0 >= p.M) return;  // uniform
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
      if (live && m < p.M) {
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
    if (row >= p.M || col >= p.N) continue;
    float v[2];
#pragma unroll
    for (int j = 0; j < NM / NT; ++j) {
      v[j] = part[0][j * NT + tile][i][at];
#pragma unroll
      for (int k = 1; k < NW; ++k) v[j] += part[k][j * NT + tile][i][at];
      if (p.bias[j]) v[j] += p.bias[j][col];
    }
    float y = v[0];
    if constexpr (GATED) y *= mx_activate(act, v[1]);
    mx_store(p.y, p.y_dt, row * p.ldy + col, y);
  }
}

template <typename X, bool FP4, bool GATED, int MT, int NT, int NW>
hipError_t launch_rows_kernel(const MxLinearParams &p, hipStream_t s) {
  const int64_t tn = (p.N + 16 * NT - 1) / (16 * NT), tm = (p.M + 16 * MT - 1) / (16 * MT), z = (tm + 65534) / 65535;  // a grid's y and z end at 65535
  if (tn * 64 * NW > UINT32_MAX || z > 65535) return hipErrorInvalidValue;  // a launch's work-items along x
  const dim3 grid((unsigned)tn, (unsigned)((tm + z - 1) / z), (unsigned)z);
  hipLaunchKernelGGL((mx_rows_kernel<X, FP4, GATED, MT, NT, NW>), grid, dim3(64 * NW), 0, s, p, mx_act(p.act));
  return hipGetLastError();
}

// us with 4 / 8 / 16 wavefronts: 1 row, 8192 -> 2048 bf16 12.9 / 8.9 / 7.4, f32
// 19.3 / 13.8 / 11.0; 2048 -> 8192 4.5 / 4.5 / 4.5, f32 6.8 / 6.4 / 6.9; 1536 ->
// 9216 5.1 / 4.8 / 5.3; 33 rows, 8192 -> 2048 23.6 / 20.4 / 20.2, 1536 -> 9216
// 13.6 / 13.0 / 14.1. Four row tiles instead of two: 64 rows, 8192 -> 2048 20.7 ->
// 35.6, 2048 -> 8192 19.9 -> 19.6. Two groups in flight a wavefront: within 8%.
template <typename X, bool FP4, bool GATED>
hipError_t launch_rows_kernel(const MxLinearParams &p, hipStream_t s) {
  if (p.M > 16) return launch_rows_kernel<X, FP4, GATED, 2, 1, 8>(p, s);
  constexpr bool two_byte = !FP4 && std::conditional_t<FP4, F32, X>::bytes == 2;
  const int nt = mx_few_tiles(two_byte, p.N, p.K, GATED);
  if constexpr (!GATED)
    if (nt == 4) return launch_rows_kernel<X, FP4, GATED, 1, 4, 8>(p, s);
  if (nt == 2) return launch_rows_kernel<X, FP4, GATED, 1, 2, 8>(p, s);
  return p.K >= 6144 ? launch_rows_kernel<X, FP4, GATED, 1, 1, 16>(p, s) : launch_rows_kernel<X, FP4, GATED, 1, 1, 8>(p, s);
}

template <typename X, bool FP4>
hipError_t launch_rows_kernel(const MxLinearParams &p, hipStream_t s) {
  return p.act >= 0 ? launch_rows_kernel<X, FP4, true>(p, s) : launch_rows_kernel<X, FP4, false>(p, s);
}

template <typename X> hipError_t launch_rows_x(const MxLinearParams &p, hipStream_t s) {
  return p.fp4 ? launch_rows_kernel<X, true>(p, s) : launch_rows_kernel<X, false>(p, s);
}

}  // namespace

hipError_t launch_mx_quantize(const MxQuantParams &p, hipStream_t s) {
  if (p.M <= 0) return hipSuccess;
  const bool two = mx_quant_tiles(p.M, p.K, 4) < 512;
  const int64_t tiles = mx_quant_tiles(p.M, p.K, two ? 2 : 4);
  if (tiles * 256 > UINT32_MAX) return hipErrorInvalidValue;  // a launch's work-items
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (two) hipLaunchKernelGGL((mx_quantize_kernel<T, 2>), dim3((unsigned)tiles), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((mx_quantize_kernel<T, 4>), dim3((unsigned)tiles), dim3(256), 0, s, p);
    return hipGetLastError();
  };
  switch (p.x_dt) {
    case LUX3D_F32: return launch(F32{});
    case LUX3D_BF16: return launch(BF16{});
    case LUX3D_F16: return launch(F16{});
  }
  return hipErrorInvalidValue;
}

hipError_t launch_mx_dequantize(const MxDequantParams &p, hipStream_t s) {
  if (p.M <= 0) return hipSuccess;
  const bool two = mx_quant_tiles(p.M, p.K, 4) < 512;
  const int64_t tiles = mx_quant_tiles(p.M, p.K, two ? 2 : 4);
  if (tiles * 256 > UINT32_MAX) return hipErrorInvalidValue;  // a launch's work-items
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (two) hipLaunchKernelGGL((mx_dequantize_kernel<T, 2>), dim3((unsigned)tiles), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((mx_dequantize_kernel<T, 4>), dim3((unsigned)tiles), dim3(256), 0, s, p);
    return hipGetLastError();
  };
  switch (p.y_dt) {
    case LUX3D_F32: return launch(F32{});
    case LUX3D_BF16: return launch(BF16{});
    case LUX3D_F16: return launch(F16{});
  }
  return hipErrorInvalidValue;
}

namespace {
hipError_t launch_rows(const MxLinearParams &p, hipStream_t s) {
  if (!p.x) return launch_rows_kernel<void, true>(p, s);
  switch (p.x_dt) {
    case LUX3D_F32: return launch_rows_x<F32>(p, s);
    case LUX3D_BF16: return launch_rows_x<BF16>(p, s);
    case LUX3D_F16: return launch_rows_x<F16>(p, s);
  }
  return hipErrorInvalidValue;
}
}  // namespace

hipError_t launch_mx_linear(const MxLinearParams &given, hipStream_t s) {
  MxLinearParams p = given;
  if (p.M <= 0 || p.N <= 0) return hipSuccess;
  if (p.fp4 && p.x && p.M > kMxFewRows) {
    const MxQuantParams q = {p.x, p.ldx, p.x_dt, p.xq, p.xs, p.M, p.K};
    if (hipError_t e = launch_mx_quantize(q, s)) return e;
    p.x = nullptr;
  }
  const MxKind kind = !p.x ? MX_PACKED : p.x_dt == LUX3D_F32 ? MX_F32 : MX_2BYTE;
  const MxChoice c = mx_choose(kind, p.M, p.N, p.K, p.act >= 0);
  if (c.rows == 0 || !mx_gemm_fits(p)) return launch_rows(p, s);
  MxLinearParams rest = p;
  p.M = c.rows;
  if (hipError_t e = launch_mx_gemm(p, c.tile, s)) return e;
  if ((rest.M -= c.rows) == 0) return hipSuccess;
  if (rest.x) rest.x = reinterpret_cast<const char *>(p.x) + c.rows * p.ldx * (p.x_dt == LUX3D_F32 ? 4 : 2);
  else rest.xq += c.rows * (p.K / 2), rest.xs += c.rows * 4;
  rest.y = reinterpret_cast<char *>(p.y) + c.rows * p.ldy * (p.y_dt == LUX3D_F32 ? 4 : 2);
  return launch_rows(rest, s);
}

}  // namespace lux3d
