// adapters.hpp -- device helpers of the low-rank adapters beside a Q8_0 linear: which rows a segment has and which
// adapter, and the second product, t B^T, added to the GEMM kernels' accumulators before their epilogues.
//
// t = alpha x A^T comes from adapter_down_kernel (adapters.hip), in x's type, rows of `tp` = rank rounded up to 16 with
// zeros behind the rank; 32 rows at a time as the fragments' lanes read it: 16-byte pieces, a piece of all 32 rows after
// the other (by rows of tp, a fragment's lanes touch 32 cache lines). For an output tile the segments that its rows fall into are taken one after the other: t's rows
// outside the segment count as zero, so that the products of several adapters add up in one accumulator.
#pragma once

#include <type_traits>

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

// Segment of `row`, the same for the whole wavefront: as segment_of has it, with one load a lane in place of a search.
__device__ __forceinline__ int64_t adapter_segment(const AdapterParams &d, int64_t row) {
  if (!d.seg_off) {
    const int64_t s = row / d.rows_per_seg;
    return s < d.nseg ? s : d.nseg - 1;
  }
  int64_t n = 0;
  for (int64_t s0 = 1; s0 < d.nseg; s0 += 64) {
    const int64_t s = s0 + (threadIdx.x & 63);
    n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(s < d.nseg && d.seg_off[s < d.nseg ? s : d.nseg] <= row));
  }
  return uniform(n);
}

// Where t holds values k .. of `row`, k a multiple of 16 / EB, and the bytes from a piece to the row's next one.
template <int EB>
__device__ __forceinline__ char *adapter_t(const AdapterParams &d, int64_t M, int64_t row, int k, int &next) {
  const int64_t tile = row >> 5;
  next = (M - tile * 32 < 32 ? (int)(M - tile * 32) : 32) * 16;
  return reinterpret_cast<char *>(d.t) + tile * 32 * d.tp * EB + (k * EB / 16) * next + (row & 31) * 16;
}
// its values k .. k + 7
__device__ __forceinline__ ad_bf16x8_t adapter_t8(const char *t, int) { return *reinterpret_cast<const ad_bf16x8_t *>(t); }
__device__ __forceinline__ void adapter_t8(const char *t, int next, float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float4 x = *reinterpret_cast<const float4 *>(t + q * next);
    v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
  }
}

// Values k .. k + 7 of B's row (zeros from the rank on), k a multiple of 8. Rows have any alignment.
__device__ __forceinline__ ad_bf16x8_t adapter_b8(const AdapterParams &d, int64_t row, int k) {
  typedef uint32_t u4_t __attribute__((ext_vector_type(4), aligned(2)));
  const uint16_t *b = reinterpret_cast<const uint16_t *>(d.b) + row * d.r + k;
  u4_t w = {0, 0, 0, 0};
  if (k + 8 <= d.r) {
    w = *reinterpret_cast<const u4_t *>(b);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = k + 2 * e < d.r ? b[2 * e] : 0, hi = k + 2 * e + 1 < d.r ? b[2 * e + 1] : 0;
      w[e] = lo | (hi << 16);
    }
  }
  return __builtin_bit_cast(ad_bf16x8_t, w);
}
__device__ __forceinline__ void adapter_b8(const AdapterParams &d, int64_t row, int k, float (&v)[8]) {
  typedef float f4_t __attribute__((ext_vector_type(4), aligned(4)));
  const float *b = reinterpret_cast<const float *>(d.b) + row * d.r + k;
#pragma unroll
  for (int h = 0; h < 8; h += 4) {
    if (k + h + 4 <= d.r) {
      const f4_t x = *reinterpret_cast<const f4_t *>(b + h);
      v[h] = x.x; v[h + 1] = x.y; v[h + 2] = x.z; v[h + 3] = x.w;
    } else {
#pragma unroll
      for (int e = h; e < h + 4; ++e) v[e] = k + e < d.r ? b[e] : 0.f;
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
//
// The GEMM kernels call it behind their first loads, so that its latency passes while those arrive. Where one segment has
// all of the rows, as most tiles do, U steps of 16 rank values are loaded together, without branches. us, the linear alone
// / with adapters added after its products / before: 9001 x 1536 -> 1536 rank 12 52 / 54.5 / 53, 4096 x 2048 -> 8192 rank
// 64 135 / 152 / 141.
template <bool XF32, int TI, int TJ>
__device__ __forceinline__ void adapter_add(const AdapterParams &d, int64_t M, int64_t N, int64_t row0, int64_t col0,
                                            ad_f32x16_t (&acc)[TI][TJ]) {
  const int lane = threadIdx.x & 63, h = lane >> 5, l32 = lane & 31;
  const int64_t end = row0 + 32 * TI < M ? row0 + 32 * TI : M;
  if (row0 >= end) return;
  int64_t s = adapter_segment(d, row0);
  int64_t hi = uniform(adapter_row(d, M, s + 1));
  int id = __builtin_amdgcn_readfirstlane(adapter_id(d, s));
  int64_t col[TJ];
#pragma unroll
  for (int j = 0; j < TJ; ++j) {
    col[j] = col0 + 32 * j + l32;
    col[j] = col[j] < N ? col[j] : N - 1;
  }
  auto run = [&](int i, const auto &a, const auto &b) {
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      if constexpr (!XF32) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
      } else {
#pragma unroll
        for (int n = 2; n >= 0; --n)  // smallest terms first: t_x b_y with x + y = n
#pragma unroll
          for (int x = 0; x <= n; ++x)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[x], b[j].t[n - x], acc[i][j], 0, 0, 0);
      }
    }
  };
  if (hi >= end) {
    if (id < 0) return;
    constexpr int EB = XF32 ? 4 : 2;
    const char *tr[TI];
    int next[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int64_t r = row0 + 32 * i + l32;
      tr[i] = adapter_t<EB>(d, M, r < end ? r : end - 1, 8 * h, next[i]);
    }
    auto steps = [&](int k, auto u_c) {
      constexpr int U = decltype(u_c)::value;
      if constexpr (!XF32) {
        ad_bf16x8_t a[U][TI], b[U][TJ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int j = 0; j < TJ; ++j) b[u][j] = adapter_b8(d, id * N + col[j], k + 16 * u + 8 * h);
#pragma unroll
          for (int i = 0; i < TI; ++i) a[u][i] = adapter_t8(tr[i] + (k / 8 + 2 * u) * next[i], next[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < TI; ++i) run(i, a[u][i], b[u]);
      } else {
        float a[U][TI][8], b[U][TJ][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int j = 0; j < TJ; ++j) adapter_b8(d, id * N + col[j], k + 16 * u + 8 * h, b[u][j]);
#pragma unroll
          for (int i = 0; i < TI; ++i) adapter_t8(tr[i] + (k / 4 + 4 * u) * next[i], next[i], a[u][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Terms3 b3[TJ];
#pragma unroll
          for (int j = 0; j < TJ; ++j) b3[j] = terms3(b[u][j]);
#pragma unroll
          for (int i = 0; i < TI; ++i) run(i, terms3(a[u][i]), b3);
        }
      }
    };
    constexpr int U = TI > 4 ? 2 : 4;
    int k = 0;
    for (; k + 16 * U <= d.tp; k += 16 * U) steps(k, std::integral_constant<int, U>{});
    if constexpr (U == 4) {
      if (k + 32 <= d.tp) {
        steps(k, std::integral_constant<int, 2>{});
        k += 32;
      }
    }
    if (k < d.tp) steps(k, std::integral_constant<int, 1>{});
    return;
  }
  // several segments: one after the other
  int64_t lo = row0;
  while (true) {
    hi = hi < end ? hi : end;
    if (id >= 0 && hi > lo) {
      for (int k = 0; k < d.tp; k += 16) {
        std::conditional_t<XF32, Terms3, ad_bf16x8_t> b[TJ];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
          if constexpr (!XF32) {
            b[j] = adapter_b8(d, id * N + col[j], k + 8 * h);
          } else {
            float v[8];
            adapter_b8(d, id * N + col[j], k + 8 * h, v);
            b[j] = terms3(v);
          }
        }
#pragma unroll
        for (int i = 0; i < TI; ++i) {
          const int64_t t0 = row0 + 32 * i, r = t0 + l32;
          if (t0 >= hi || t0 + 32 <= lo) continue;  // uniform
          const bool in = r >= lo && r < hi;
          int next;
          const char *at = adapter_t<XF32 ? 4 : 2>(d, M, in ? r : lo, k + 8 * h, next);
          if constexpr (!XF32) {
            ad_bf16x8_t a = __builtin_bit_cast(ad_bf16x8_t, make_uint4(0, 0, 0, 0));
            if (in) a = adapter_t8(at, next);
            run(i, a, b);
          } else {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
            if (in) adapter_t8(at, next, v);
            run(i, terms3(v), b);
          }
        }
      }
    }
    lo = hi > lo ? hi : lo;
    if (lo >= end || ++s >= d.nseg) break;
    hi = uniform(adapter_row(d, M, s + 1));
    id = __builtin_amdgcn_readfirstlane(adapter_id(d, s));
  }
}

// t B^T of one output (row, col), for kernels that hold single outputs
template <bool XF32>
__device__ __forceinline__ float adapter_dot(const AdapterParams &d, int64_t M, int64_t N, int64_t row, int64_t col) {
  const int id = adapter_id(d, segment_of(d.seg_off, d.nseg, d.rows_per_seg, row));
  if (id < 0) return 0.f;
  float acc = 0.f;
  for (int k = 0; k < d.tp; k += 8) {
    float t[8], b[8];
    int next;
    const char *at = adapter_t<XF32 ? 4 : 2>(d, M, row, k, next);
    if constexpr (XF32) {
      adapter_t8(at, next, t);
      adapter_b8(d, id * N + col, k, b);
    } else {
      Chunk<BF16>::load<false>(at, t);
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
