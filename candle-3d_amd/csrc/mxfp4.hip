// mxfp4.hip -- microscaled 4-bit values on gfx950: quantisation, its inverse,
// and the linear layers of few rows (mxfp4.hpp: the format).
#include "mxfp4_rows.hpp"

namespace lux3d {

namespace {

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
//
// COLS: rows of up to 128 and 256 values share a wavefront's 512, 4 and 2 at a time
// (100000 rows, us, a row a wavefront / shared: 128 bf16 12.1 / 7.7, 64 f32 12.5 /
// 8.2, 256 bf16 14.7 / 13.6; back 7.1 / 5.5, 7.0 / 5.5, 11.1 / 11.0).
inline int mx_quant_cols(int64_t k) { return k <= 128 ? 128 : k <= 256 ? 256 : 512; }
inline int64_t mx_quant_tiles(int64_t rows, int64_t k, int r) {
  const int64_t cols = mx_quant_cols(k), tile = 4 * r * 512 / cols;
  return (k + cols - 1) / cols * ((rows + tile - 1) / tile);
}

template <typename T, int R, int COLS>
__global__ __launch_bounds__(256) void mx_quantize_kernel(MxQuantParams p) {
  constexpr int NV = T::bytes == 4 ? 2 : 1;  // 16-byte loads a lane and row
  constexpr int L = COLS / 8, RL = 64 / L, ROWS = 4 * R * RL;  // lanes of a row; rows of a load, of the workgroup
  __shared__ uint32_t sc[COLS / 128][ROWS];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t tk = (p.K + COLS - 1) / COLS, rt = (int64_t)blockIdx.x / tk, kt = blockIdx.x - rt * tk;
  const int64_t r0 = rt * ROWS, k = kt * COLS + lane % L * 8;
  const int lr = wave * R * RL + lane / L;  // row of the workgroup, of the lane's first
  const bool live = k < p.K;
  uint32_t v[R][4 * NV];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int64_t r = r0 + lr + i * RL;
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
    const int64_t r = r0 + lr + i * RL;
    uint32_t top = mx_top<T>(v[i]);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, DPP_XOR1, 0xF, 0xF, false));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, DPP_XOR2, 0xF, 0xF, false));
    const uint32_t s = mx_scale(top);  // values past K count as 0: so do the scales that fill up the last group
    const uint32_t codes = mx_codes<T>(v[i], s);
    if (live && r < p.M) *reinterpret_cast<uint32_t *>(p.q + (r * p.K + k) / 2) = codes;
    if ((lane & 3) == 0) reinterpret_cast<uint8_t *>(&sc[lane % L >> 4][lr + i * RL])[(lane >> 2) & 3] = (uint8_t)s;
  }
  __syncthreads();
  const int64_t g = kt * (COLS / 128) + t / ROWS, r = r0 + t % ROWS;
  if (t < 16 * R && g * 128 < p.K && r < p.M) reinterpret_cast<uint32_t *>(p.s)[g * p.M + r] = sc[t / ROWS][t % ROWS];
}

// ---- and back -------------------------------------------------------------------
//
// The same tiles, R rows of a wavefront in flight. A lane writes 16 bytes and the
// next lane the 16 behind them: 8 values of a 2-byte type, 4 of f32, which takes
// the row's half in two steps (16 values a lane and four stores 64 bytes apart
// instead: 8192 x 2048 f32 50 us against 12).
template <typename T, int R, int COLS>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxDequantParams p) {
  constexpr int V = 16 / T::bytes, STEPS = 8 / V, L = COLS / 8, RL = 64 / L;  // values a lane and step; lanes of a row; rows of a store
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t tk = (p.K + COLS - 1) / COLS, rt = (int64_t)blockIdx.x / tk, kt = blockIdx.x - rt * tk;
  const int64_t r0 = rt * (4 * R * RL) + wave * R * RL + lane / L;
#pragma unroll
  for (int step = 0; step < STEPS; ++step) {
    const int64_t k = kt * COLS + step * (COLS / STEPS) + lane % L * V;
    if (k >= p.K) return;
    uint32_t c[R], s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i * RL < p.M ? r0 + i * RL : p.M - 1;
      const uint8_t *src = p.q + (r * p.K + k) / 2;
      if constexpr (V == 8) c[i] = *reinterpret_cast<const uint32_t *>(src);
      else c[i] = *reinterpret_cast<const uint16_t *>(src);
      s[i] = p.s[((k >> 7) * p.M + r) * 4 + ((k >> 5) & 3)];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (r0 + i * RL >= p.M) break;
      void *dst = reinterpret_cast<char *>(p.y) + ((r0 + i * RL) * p.ldy + k) * T::bytes;
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

template <typename X, bool FP4, bool GATED, int MT, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void mx_rows_kernel(MxLinearParams p, MxAct act) {
  __shared__ float lds[mx_rows_lds<GATED, MT, NT, NW> / 4];
  const int64_t m0 = ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * 16 * MT;
  if (m0 < p.M) mx_rows_tile<X, FP4, GATED, MT, NT, NW>(p, act, m0, p.M, (int64_t)blockIdx.x * 16 * NT, lds);  // uniform
}

template <typename X, bool FP4, bool GATED, int MT, int NT, int NW>
hipError_t launch_rows_kernel(const MxLinearParams &p, hipStream_t s) {
  const int64_t tn = (p.N + 16 * NT - 1) / (16 * NT), tm = (p.M + 16 * MT - 1) / (16 * MT), z = (tm + 65534) / 65535;  // a grid's y and z end at 65535
  if (tn * 64 * NW > UINT32_MAX || z > 65535) return hipErrorInvalidValue;  // a launch's work-items along x
  const dim3 grid((unsigned)tn, (unsigned)((tm + z - 1) / z), (unsigned)z);
  hipLaunchKernelGGL((mx_rows_kernel<X, FP4, GATED, MT, NT, NW>), grid, dim3(64 * NW), 0, s, p, mx_act(p.act));
  return hipGetLastError();
}

template <typename X, bool FP4, bool GATED>
hipError_t launch_rows_kernel(const MxLinearParams &p, hipStream_t s) {
  constexpr bool two_byte = !FP4 && std::conditional_t<FP4, F32, X>::bytes == 2;
  const MxFewTile f = mx_few_tile(two_byte, p.M, p.N, p.K, GATED);
  const auto is = [&](int rows, int cols, int waves) { return f.rows == rows && f.cols == cols && f.waves == waves; };
  if constexpr (!FP4 || std::is_void_v<X>)  // more rows that enter in 4 bits are packed before
    if (is(2, 1, 8)) return launch_rows_kernel<X, FP4, GATED, 2, 1, 8>(p, s);
  if (is(1, 1, 8)) return launch_rows_kernel<X, FP4, GATED, 1, 1, 8>(p, s);
  if (is(1, 1, 16)) return launch_rows_kernel<X, FP4, GATED, 1, 1, 16>(p, s);
  if (is(1, 2, 8)) return launch_rows_kernel<X, FP4, GATED, 1, 2, 8>(p, s);
  if constexpr (!GATED)
    if (is(1, 4, 8)) return launch_rows_kernel<X, FP4, GATED, 1, 4, 8>(p, s);
  return hipErrorInvalidValue;
}

template <typename X, bool FP4>
hipError_t launch_rows_kernel(const MxLinearParams &p, hipStream_t s) {
  return p.act >= 0 ? launch_rows_kernel<X, FP4, true>(p, s) : launch_rows_kernel<X, FP4, false>(p, s);
}

template <typename X> hipError_t launch_rows_x(const MxLinearParams &p, hipStream_t s) {
  return p.fp4 ? launch_rows_kernel<X, true>(p, s) : launch_rows_kernel<X, false>(p, s);
}

}  // namespace

namespace {
template <int I> using int_t = std::integral_constant<int, I>;
template <typename F> hipError_t mx_quant_variant(bool two, int64_t k, F with) {
  switch (mx_quant_cols(k)) {
    case 128: return two ? with(int_t<2>{}, int_t<128>{}) : with(int_t<4>{}, int_t<128>{});
    case 256: return two ? with(int_t<2>{}, int_t<256>{}) : with(int_t<4>{}, int_t<256>{});
  }
  return two ? with(int_t<2>{}, int_t<512>{}) : with(int_t<4>{}, int_t<512>{});
}
}  // namespace

hipError_t launch_mx_quantize(const MxQuantParams &p, hipStream_t s) {
  if (p.M <= 0) return hipSuccess;
  const bool two = mx_quant_tiles(p.M, p.K, 4) < 512;
  const int64_t tiles = mx_quant_tiles(p.M, p.K, two ? 2 : 4);
  if (tiles * 256 > UINT32_MAX) return hipErrorInvalidValue;  // a launch's work-items
  auto launch = [&](auto type) {
    using T = decltype(type);
    auto with = [&](auto rows, auto cols) {
      hipLaunchKernelGGL((mx_quantize_kernel<T, decltype(rows)::value, decltype(cols)::value>), dim3((unsigned)tiles), dim3(256), 0, s, p);
      return hipGetLastError();
    };
    return mx_quant_variant(two, p.K, with);
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
    auto with = [&](auto rows, auto cols) {
      hipLaunchKernelGGL((mx_dequantize_kernel<T, decltype(rows)::value, decltype(cols)::value>), dim3((unsigned)tiles), dim3(256), 0, s, p);
      return hipGetLastError();
    };
    return mx_quant_variant(two, p.K, with);
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
  if (c.rows == 0 || !mx_gemm_fits(kind, p.ldx, p.xs_rows, p.N, p.K, p.ldy)) return launch_rows(p, s);
  p.rest = p.M - c.rows;
  p.M = c.rows;
  return launch_mx_gemm(p, c.tile, s);
}

}  // namespace lux3d
