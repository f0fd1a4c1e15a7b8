// adapters.hpp -- device helpers of the low-rank adapters beside a Q8_0 linear: which rows a segment has and which
// adapter, and the second product, t B^T, added to the GEMM kernels' accumulators before their epilogues.
//
// t = alpha x A^T comes from adapter_down_kernel (adapters.hip), in x's type, rows of `tp` = rank rounded up to 16 with
// zeros behind the rank. For an output tile the segments that its rows fall into are taken one after the other: t's rows
// outside the segment count as zero, so that the products of several adapters add up in one accumulator.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace lux3d {

typedef __bf16 ad_bf16x8_t __attribute__((ext_vector_type(8)));
typedef float ad_f32x16_t __attribute__((ext_vector_type(16)));

// First row of segment s (s up to nseg): rows before the first offset are segment 0's, rows from the last one on the
// last segment's, as segment_of has it.
__device__ __forceinline__ int64_t adapter_row(const AdapterParams &d, int64_t rows, int64_t s) {
  if (s <= 0) return 0;
  if (s >= d.nseg) return rows;
  int64_t r = d.seg_off ? d.seg_off[s] : s * d.rows_per_seg;
  r = r < 0 ? 0 : r;
  return r < rows ? r : rows;
}
// The segment's adapter, -1 for none.
__device__ __forceinline__ int adapter_id(const AdapterParams &d, int64_t s) {
  const int id = d.ids[s];
  return id >= 0 && id < d.n ? id : -1;
}

// Values k .. k + 7 of B's row (zeros from the rank on), k a multiple of 8.
__device__ __forceinline__ ad_bf16x8_t adapter_b8(const AdapterParams &d, int64_t row, int k) {
  const uint16_t *b = reinterpret_cast<const uint16_t *>(d.b) + row * d.r;
  if (d.b_vec) {
    if (k >= d.r) return __builtin_bit_cast(ad_bf16x8_t, make_uint4(0, 0, 0, 0));
    return *reinterpret_cast<const ad_bf16x8_t *>(b + k);
  }
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = k + 2 * e < d.r ? b[k + 2 * e] : 0, hi = k + 2 * e + 1 < d.r ? b[k + 2 * e + 1] : 0;
    w[e] = lo | (hi << 16);
  }
  return __builtin_bit_cast(ad_bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void adapter_b8(const AdapterParams &d, int64_t row, int k, float (&v)[8]) {
  const float *b = reinterpret_cast<const float *>(d.b) + row * d.r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (d.b_vec) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k + 4 * h < d.r) x = *reinterpret_cast<const float4 *>(b + k + 4 * h);
      v[4 * h] = x.x; v[4 * h + 1] = x.y; v[4 * h + 2] = x.z; v[4 * h + 3] = x.w;
    } else {
#pragma unroll
      for (int e = 4 * h; e < 4 * h + 4; ++e) v[e] = k + e < d.r ? b[k + e] : 0.f;
    }
  }
}

struct Terms3 {
  ad_bf16x8_t t[3];
};
__device__ __forceinline__ Terms3 terms3(const float (&v)[8]) {
  uint32_t w[3][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const Split3 s = split3_bf16(v[2 * e], v[2 * e + 1]);
    w[0][e] = s.t1;
    w[1][e] = s.t2;
    w[2][e] = s.t3;
  }
  Terms3 r;
#pragma unroll
  for (int i = 0; i < 3; ++i) r.t[i] = __builtin_bit_cast(ad_bf16x8_t, make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]));
  return r;
}

// acc[i][j] += t B^T for the wavefront's TI x TJ tiles of 32 x 32: rows row0 + 32 i, columns col0 + 32 j. All of the
// tile's rows and columns past the matrix are computed from clamped addresses and never stored. XF32: t and B are f32, in
// three exact bf16 terms each and the six significant products, as the f32 GEMM has it.
template <bool XF32, int TI, int TJ>
__device__ __forceinline__ void adapter_add(const AdapterParams &d, int64_t M, int64_t N, int64_t row0, int64_t col0,
                                            ad_f32x16_t (&acc)[TI][TJ]) {
  const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
  const int64_t end = row0 + 32 * TI < M ? row0 + 32 * TI : M;
  if (row0 >= end) return;
  int64_t col[TJ];
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    col[j] = col0 + 32 * j + l32;
    col[j] = col[j] < N ? col[j] : N - 1;
  }
  int64_t s = uniform(segment_of(d.seg_off, d.nseg, d.rows_per_seg, row0));
  int64_t lo = row0;
  while (lo < end) {
    int64_t hi = uniform(adapter_row(d, M, s + 1));
    const int id = __builtin_amdgcn_readfirstlane(adapter_id(d, s));
    hi = hi < end ? hi : end;
    if (id >= 0 && hi > lo) {
      for (int k = 0; k < d.tp; k += 16) {
        if constexpr (!XF32) {
          ad_bf16x8_t b[TJ];
#pragma unroll
          for (int j = 0; j < TJ; ++j) b[j] = adapter_b8(d, id * N + col[j], k + 8 * h);
#pragma unroll
          for (int i = 0; i < TI; ++i) {
            const int64_t t0 = row0 + 32 * i, r = t0 + l32;
            if (t0 >= hi || t0 + 32 <= lo) continue;  // uniform
            uint4 a = make_uint4(0, 0, 0, 0);
            if (r >= lo && r < hi) a = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(d.t) + r * d.tp + k + 8 * h);
#pragma unroll
            for (int j = 0; j < TJ; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ad_bf16x8_t, a), b[j], acc[i][j], 0, 0, 0);
          }
        } else {
          Terms3 b[TJ];
#pragma unroll
          for (int j = 0; j < TJ; ++j) {
            float v[8];
            adapter_b8(d, id * N + col[j], k + 8 * h, v);
            b[j] = terms3(v);
          }
#pragma unroll
          for (int i = 0; i < TI; ++i) {
            const int64_t t0 = row0 + 32 * i, r = t0 + l32;
            if (t0 >= hi || t0 + 32 <= lo) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
            if (r >= lo && r < hi) Chunk<F32>::load<false>(reinterpret_cast<const float *>(d.t) + r * d.tp + k + 8 * h, v);
            const Terms3 a = terms3(v);
#pragma unroll
            for (int j = 0; j < TJ; ++j)
#pragma unroll
              for (int n = 2; n >= 0; --n)  // smallest terms first: t_x b_y with x + y = n
#pragma unroll
                for (int x = 0; x <= n; ++x)
                  acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[x], b[j].t[n - x], acc[i][j], 0, 0, 0);
          }
        }
      }
    }
    lo = hi > lo ? hi : lo;
    if (++s >= d.nseg) break;
  }
}

// t B^T of one output (row, col), for kernels that hold single outputs
template <bool XF32>
__device__ __forceinline__ float adapter_dot(const AdapterParams &d, int64_t N, int64_t row, int64_t col) {
  const int id = adapter_id(d, segment_of(d.seg_off, d.nseg, d.rows_per_seg, row));
  if (id < 0) return 0.f;
  float acc = 0.f;
  for (int k = 0; k < d.tp; k += 8) {
    float t[8], b[8];
    if constexpr (XF32) {
      Chunk<F32>::load<false>(reinterpret_cast<const float *>(d.t) + row * d.tp + k, t);
      adapter_b8(d, id * N + col, k, b);
    } else {
      Chunk<BF16>::load<false>(reinterpret_cast<const uint16_t *>(d.t) + row * d.tp + k, t);
      const uint4 w = __builtin_bit_cast(uint4, adapter_b8(d, id * N + col, k));
      const uint32_t w4[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = bf16_bits_to_f32((w4[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_fmaf(t[e], b[e], acc);
  }
  return acc;
}

}  // namespace lux3d
