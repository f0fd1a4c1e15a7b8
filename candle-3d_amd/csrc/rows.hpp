// rows.hpp -- device helpers of the row kernels (norm_rows.hip, block_norm.hip):
// a row's chunks and their 16-byte accesses, its parameters, its segment and
// the sums over it.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace lux3d {

constexpr int kBlock = 256;

// Segment of row r: the launcher's magic division for dense segments, the
// scalar binary search over the offsets for ragged ones.
__device__ __forceinline__ int64_t row_segment(const RowParams &p, int64_t r) {
  if (p.rps_m) return segment_of_dense((uint32_t)r, p.rps_m, p.rps_s, p.nseg);
  return segment_of(p.seg_off, p.nseg, p.rows_per_seg, r);
}

template <int TPR, int BLOCK = kBlock>
__device__ __forceinline__ float row_total(float s, float *red) {
  s = wave_sum(s);
  if constexpr (TPR == 64) {
    return s;
  } else {
    constexpr int WPR = TPR / 64;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = s;
    lds_barrier();  // the row's stores (e.g. the residual stream h) stay in flight
    const int w0 = (w / WPR) * WPR;
    float tot = red[w0];
#pragma unroll
    for (int k = 1; k < WPR; ++k) tot += red[w0 + k];
    return tot;
  }
}

// Element offsets of chunk c of lane t in a row: its two 4-element halves.
// 2-byte types: 8 consecutive elements (one 16-byte access). f32: the halves
// lie TPR * 4 elements apart, so that every 16-byte access instruction of a
// wavefront covers 1 KiB of contiguous row (32 consecutive bytes per lane
// would make each instruction touch 2 KiB with half of it used; the copy
// of that layout measured 12-16% slower than the interleaved one at the
// configs' f32 rows). The row's statistics do not depend on which elements a
// lane holds, and every operand of an element uses the same offsets.
struct ChunkAt {
  int64_t o0, o1;
};
template <typename T, int TPR>
__device__ __forceinline__ ChunkAt chunk_at(int c, int t) {
  if constexpr (T::bytes == 4) return {(int64_t)(2 * c * TPR + t) * 4, (int64_t)((2 * c + 1) * TPR + t) * 4};
  else return {(int64_t)(c * TPR + t) * 8, (int64_t)(c * TPR + t) * 8 + 4};
}
template <typename T>
__device__ __forceinline__ void ld_row(const char *row, ChunkAt a, float (&v)[8]) {
  if constexpr (T::bytes == 4) {
    const uint4 x = ld16<LUX3D_NT_STREAMS != 0>(row + a.o0 * 4), y = ld16<LUX3D_NT_STREAMS != 0>(row + a.o1 * 4);
    v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
    v[4] = __uint_as_float(y.x); v[5] = __uint_as_float(y.y); v[6] = __uint_as_float(y.z); v[7] = __uint_as_float(y.w);
  } else {
    Chunk<T>::load(row + a.o0 * T::bytes, v);
  }
}
template <typename T>
__device__ __forceinline__ void st_row(char *row, ChunkAt a, const float (&v)[8]) {
  if constexpr (T::bytes == 4) {
    st16(row + a.o0 * 4, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                    __float_as_uint(v[3])));
    st16(row + a.o1 * 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]),
                                    __float_as_uint(v[7])));
  } else {
    Chunk<T>::store(row + a.o0 * T::bytes, v);
  }
}
// the parameters of chunk a (offset by off elements)
template <typename T>
__device__ __forceinline__ void param_at(const void *p, int dt, int64_t off, ChunkAt a, float dflt, float (&v)[8]) {
  if constexpr (T::bytes == 4) {
    param4(p, dt, off + a.o0, dflt, v);
    param4(p, dt, off + a.o1, dflt, v + 4);
  } else {
    param8(p, dt, off + a.o0, dflt, v);
  }
}
template <typename T>
__device__ __forceinline__ void mod_at(const ModPiece &m, int64_t seg, ChunkAt a, float dflt, float (&v)[8]) {
  param_at<T>(m.p, m.dt, seg * m.ld, a, dflt, v);
  if (m.base_dt >= 0) {
    float b[8];
    param_at<T>(m.base, m.base_dt, 0, a, 0.f, b);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = b[k] + v[k];
  }
}
__device__ __forceinline__ void lds_at(const float *src, ChunkAt a, float (&v)[8]) {
  const float4 x = *reinterpret_cast<const float4 *>(src + a.o0);
  const float4 y = *reinterpret_cast<const float4 *>(src + a.o1);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}

}  // namespace lux3d
