// adapters.hip -- the first product of the low-rank adapters beside a Q8_0 linear: t = alpha x A^T for rows whose
// segment has an adapter (the second, t B^T, is added in the GEMM's epilogue, adapters.hpp).
//
// x's bytes bound it, or for few rows A's. A workgroup takes 16 rows of one segment and 16 NT values of the rank; its
// wavefronts take 64-deep chunks of k in turn and their sums are added in wavefront order through LDS
// (v_mfma_f32_16x16x32_bf16, f32 sums; f32 x: v_mfma_f32_16x16x4_f32). t is rounded once to x's type, as an activation
// between two linear layers is.
#include "adapters.hpp"

namespace lux3d {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Tile `tile` of 16 rows within segments: its segment and first row, or s = nseg past the last one. Every lane of the
// wavefront calls it; lanes take one segment each.
struct AdapterTile {
  int64_t s, row;
};
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterParams &d, int64_t rows, int64_t tile) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int64_t s0 = 0; s0 < d.nseg; s0 += 64) {
    const int64_t s = s0 + lane, a = adapter_row(d, rows, s), b = s < d.nseg ? adapter_row(d, rows, s + 1) : a;
    int64_t n = b > a ? (b - a + 15) / 16 : 0, sum = n;
    if (s >= d.nseg) sum = n = 0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int64_t o = __shfl_up(sum, m, 64);
      if (lane >= m) sum += o;
    }
    // the first segment whose tiles reach past `tile`
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > tile);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int64_t first = before + __shfl(sum, at, 64) - __shfl(n, at, 64);
      return {uniform(s0 + at), uniform(__shfl(a, at, 64) + (tile - first) * 16)};
    }
    before += uniform(__shfl(sum, 63, 64));
  }
  return {d.nseg, 0};
}

template <bool XF32, int NT, int NW>
__global__ __launch_bounds__(64 * NW) void adapter_down_kernel(AdapterDownParams p) {
  constexpr int EB = XF32 ? 4 : 2;
  __shared__ float part[NW][NT * 256];
  const AdapterParams &d = p.ad;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4, l16 = lane & 15;
  const int j0 = (int)blockIdx.y * 16 * NT;
  if (p.bad && blockIdx.x == 0 && blockIdx.y == 0 && wave == 0) {
    // segments whose id is neither -1 nor an adapter's
    int bad = 0;
    for (int64_t s = lane; s < d.nseg; s += 64) bad += d.ids[s] < -1 || d.ids[s] >= d.n;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) bad += __shfl_xor(bad, m, 64);
    if (lane == 0) *p.bad = bad;
  }
  const AdapterTile w = adapter_tile(d, p.M, blockIdx.x);
  if (w.s >= d.nseg) return;  // uniform over the workgroup, as all that follows
  const int id = __builtin_amdgcn_readfirstlane(adapter_id(d, w.s));
  if (id < 0) return;
  const int64_t end = uniform(adapter_row(d, p.M, w.s + 1));
  // rows past the segment are clamped: loaded, computed, never stored; so are values past the rank
  const int64_t row = w.row + l16 < end ? w.row + l16 : end - 1;
  const char *xr = reinterpret_cast<const char *>(p.x) + row * p.ldx * EB;
  const char *ar[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int j = j0 + 16 * n + l16;
    ar[n] = reinterpret_cast<const char *>(d.a) + ((int64_t)id * d.r + (j < d.r ? j : d.r - 1)) * p.K * EB;
  }
  f32x4_t acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = f32x4_t{};
  // chunk c: values 64 c .. + 63; lane group g holds 16 g .. + 15 of them on both operands
  const int64_t nch = p.K / 64;
  for (int64_t c = wave; c < nch; c += NW) {
    if constexpr (!XF32) {
      const int64_t at = (c * 64 + 16 * g) * 2;
      const uint4 x0 = ld16<false>(xr + at), x1 = ld16<false>(xr + at + 16);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 a0 = ld16<false>(ar[n] + at), a1 = ld16<false>(ar[n] + at + 16);
        acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8_t, x0), __builtin_bit_cast(ad_bf16x8_t, a0), acc[n], 0, 0, 0);
        acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8_t, x1), __builtin_bit_cast(ad_bf16x8_t, a1), acc[n], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t at = (c * 64 + 16 * g + 4 * q) * 4;
        const float4 x = *reinterpret_cast<const float4 *>(xr + at);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 a = *reinterpret_cast<const float4 *>(ar[n] + at);
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, a.x, acc[n], 0, 0, 0);
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, a.y, acc[n], 0, 0, 0);
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, a.z, acc[n], 0, 0, 0);
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, a.w, acc[n], 0, 0, 0);
        }
      }
    }
  }
  if (p.K % 64 && wave == (int)(nch % NW)) {
    // the last 32 values (bf16 alone): 8 a lane group
    const int64_t at = (nch * 64 + 8 * g) * 2;
    if constexpr (!XF32) {
      const uint4 x0 = ld16<false>(xr + at);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 a0 = ld16<false>(ar[n] + at);
        acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8_t, x0), __builtin_bit_cast(ad_bf16x8_t, a0), acc[n], 0, 0, 0);
      }
    }
  }
  // lane holds rows 4 g + e, rank value lane % 16 of each tile
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][n * 256 + e * 64 + lane] = acc[n][e];
  __syncthreads();
  const float alpha = d.alpha ? d.alpha[id] : 1.f;
  for (int o = t; o < NT * 256; o += 64 * NW) {
    const int64_t r = w.row + 4 * ((o & 63) >> 4) + (o >> 6 & 3);
    const int j = j0 + (o >> 8) * 16 + (o & 15);
    if (r >= end || j >= d.tp) continue;
    float v = part[0][o];
#pragma unroll
    for (int k = 1; k < NW; ++k) v += part[k][o];
    v = j < d.r ? v * alpha : 0.f;
    if constexpr (XF32) reinterpret_cast<float *>(d.t)[r * d.tp + j] = v;
    else store1<BF16>(d.t, r * d.tp + j, v);
  }
}

template <bool XF32>
hipError_t launch_down(const AdapterDownParams &p, hipStream_t s) {
  const AdapterParams &d = p.ad;
  // at most one partly filled tile a segment
  int64_t tiles = p.M / 16 + d.nseg;
  tiles = tiles < p.M ? tiles : p.M;
  if (tiles > INT32_MAX) return hipErrorInvalidValue;
  const int nt = d.tp <= 16 ? 1 : d.tp <= 32 ? 2 : 4;
  const dim3 grid((unsigned)tiles, (unsigned)((d.tp + 16 * nt - 1) / (16 * nt)));
  if (nt == 1) hipLaunchKernelGGL((adapter_down_kernel<XF32, 1, 8>), grid, dim3(512), 0, s, p);
  else if (nt == 2) hipLaunchKernelGGL((adapter_down_kernel<XF32, 2, 8>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((adapter_down_kernel<XF32, 4, 8>), grid, dim3(512), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_adapter_down(const AdapterDownParams &p, bool x_f32, hipStream_t s) {
  if (p.M <= 0) return hipSuccess;
  return x_f32 ? launch_down<true>(p, s) : launch_down<false>(p, s);
}

}  // namespace lux3d
