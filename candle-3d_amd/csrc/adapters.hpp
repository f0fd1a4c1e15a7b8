// adapters.hpp -- device helpers of the low-rank adapters beside a Q8_0 linear: which rows a segment has and which
// adapter, and the second product, t B^T, in which the GEMM kernels' accumulators begin.
//
// t = alpha x A^T comes from adapter_down_kernel (adapters.hip), in x's type, rows of `tp` = rank rounded up to 16 with
// zeros behind the rank; 32 rows at a time as the fragments' lanes read it: 16-byte pieces, a piece of all 32 rows after
// the other (by rows of tp, a fragment's lanes touch 32 cache lines).
#pragma once

#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace lux3d {

typedef __bf16 ad_bf16x8_t __attribute__((ext_vector_type(8)));
typedef float ad_f32x4_t __attribute__((ext_vector_type(4)));
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

// Segment of `row`, the same for the whole wavefront: as segment_of has it, up to 65 segments with one load a lane in place
// of a search.
__device__ __forceinline__ int64_t adapter_segment(const AdapterParams &d, int64_t row) {
  if (!d.seg_off || d.nseg > 65) return uniform(segment_of(d.seg_off, d.nseg, d.rows_per_seg, row));
  const int64_t s = (threadIdx.x & 63) + 1;
  return __builtin_popcountll(__builtin_amdgcn_ballot_w64(s < d.nseg && d.seg_off[s < d.nseg ? s : d.nseg] <= row));
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
  } else if (k < d.r) {  // the row's last d.r % 8 values
    typedef uint32_t u1_t __attribute__((aligned(2)));
    const int n = d.r & 7;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n >= 2 * e + 2) w[e] = reinterpret_cast<const u1_t *>(b)[e];
      else if (n == 2 * e + 1) w[e] = b[2 * e];
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
      for (int e = h; e < h + 4; ++e) v[e] = 0.f;
      if (k + h < d.r) {
#pragma unroll
        for (int e = h; e < h + 3; ++e)
          if (k + e < d.r) v[e] = b[e];
      }
    }
  }
}

// The adapters of a tile's rows, row0 + 32 i + lane % 32, and the walk over them: each adapter once, whatever segments have
// it, 16 values of the rank a step (next) or all of them (next_adapter). The same for the whole wavefront.
template <int TI>
struct AdapterWalk {
  static constexpr int kBits = 0x7FFFFFFF;
  const AdapterParams &d;
  int rid[TI];       // the row's adapter, with the sign bit set once it had its turn; -1: none
  int adapter = 0;   // this step's, an adapter past the last step, too
  int who = -2;      // the same; no row's then
  int k = 1 << 30;   // its first rank value

  __device__ __forceinline__ AdapterWalk(const AdapterParams &d_, int64_t M, int64_t row0, int64_t last, int64_t s0) : d(d_) {
    const int lane = threadIdx.x & 63, r = lane & 31;
#pragma unroll
    for (int i = 0; i < TI; ++i) rid[i] = -1;
    for (; s0 < d.nseg; s0 += 64) {
      const int64_t s = s0 + lane;
      int64_t from = last, to = last;
      int id = -1;
      if (s < d.nseg) {
        from = adapter_row(d, M, s);
        to = adapter_row(d, M, s + 1);
        id = adapter_id(d, s);
      }
      const int lo = (int)((from > row0 ? from < last ? from : last : row0) - row0);
      const int hi = (int)((to < last ? to > row0 ? to : row0 : last) - row0);
      for (uint64_t mask = __builtin_amdgcn_ballot_w64(hi > lo && id >= 0); mask; mask &= mask - 1) {
        const int of = __builtin_ctzll(mask);
        const int first = __builtin_amdgcn_readlane(lo, of), end = __builtin_amdgcn_readlane(hi, of);
        const int a = __builtin_amdgcn_readlane(id, of);
#pragma unroll
        for (int i = 0; i < TI; ++i)
          if (32 * i + r >= first && 32 * i + r < end) rid[i] = a;
      }
      if (!(__builtin_amdgcn_ballot_w64(from < last) >> 63)) break;  // the next segments lie past the tile
    }
  }
  // To the next step; false past the last one. Not to be called after that.
  __device__ __forceinline__ bool next() {
    k += 16;
    return k < d.tp || next_adapter();
  }
  __device__ __forceinline__ bool next_adapter() {
    k = 0;
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const uint64_t left = __builtin_amdgcn_ballot_w64(rid[i] >= 0);
      if (!left) continue;  // uniform
      who = adapter = __builtin_amdgcn_readlane(rid[i], __builtin_ctzll(left));
#pragma unroll
      for (int j = 0; j < TI; ++j)
        if (rid[j] == adapter) rid[j] |= ~kBits;
      return true;
    }
    who = -2;
    return false;
  }
  __device__ __forceinline__ bool has(int i, int of) const { return (rid[i] & kBits) == of; }
};

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

// Eight values of an operand as they are loaded, and as the matrix instructions take them.
struct Values8 {
  float v[8];
};
__device__ __forceinline__ ad_bf16x8_t adapter_terms(ad_bf16x8_t x) { return x; }
__device__ __forceinline__ Terms3 adapter_terms(const Values8 &x) { return terms3(x.v); }
template <bool XF32>
__device__ __forceinline__ auto adapter_b(const AdapterParams &d, int64_t row, int k) {
  if constexpr (!XF32) {
    return adapter_b8(d, row, k);
  } else {
    Values8 x;
    adapter_b8(d, row, k, x.v);
    return x;
  }
}
// t's values k .. k + 7 of `row` if `in`, else zeros
template <bool XF32>
__device__ __forceinline__ auto adapter_t_row(const AdapterParams &d, int64_t M, int64_t row, bool in, int k) {
  int next;
  std::conditional_t<XF32, Values8, ad_bf16x8_t> x = {};
  if (in) {
    const char *at = adapter_t<XF32 ? 4 : 2>(d, M, row, k, next);
    if constexpr (!XF32) x = adapter_t8(at, next);
    else adapter_t8(at, next, x.v);
  }
  return x;
}

// acc[i][j] += t B^T for the wavefront's TI x TJ tiles of 32 x 32: rows row0 + 32 i, columns col0 + 32 j. All of the
// tile's rows and columns past the matrix are computed from clamped addresses and never stored. XF32: t and B are f32, in
// three exact bf16 terms each and the six significant products, as the f32 GEMM has it.
//
// The GEMM kernels call it behind their first loads, so that its latency passes while those arrive. Where one segment has
// all of the rows, as most tiles do, U steps of 16 rank values are loaded together, without branches. Other tiles go adapter
// by adapter and row tile by row tile; picking a product's rows costs 48 instructions a row tile, hence once an adapter and
// not once a step (4096 rows below: 159 us). us, the kernel alone / with adapters (shortest of 30): 9001 x 1536 -> 1536 of
// rank 12, 24 segments 53 / 57; 4096 x 2048 -> 8192 of rank 64, 4 segments 135 / 149; 3087 x 4096 -> 1024 f32 of rank 32
// 141 / 148; 12 x 1536 -> 9216 of rank 16, a segment a row 6.6 / 9.4.
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
  auto run = [&](ad_f32x16_t (&to)[TJ], const auto &a, const auto &b) {
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      if constexpr (!XF32) {
        to[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], to[j], 0, 0, 0);
      } else {
#pragma unroll
        for (int n = 2; n >= 0; --n)  // smallest terms first: t_x b_y with x + y = n
#pragma unroll
          for (int x = 0; x <= n; ++x)
            to[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.t[x], b[j].t[n - x], to[j], 0, 0, 0);
      }
    }
  };
  if (hi >= end && row0 + 32 * TI <= M && row0 % 32 == 0) {
    if (id < 0) return;
    constexpr int EB = XF32 ? 4 : 2;
    // whole groups of 32 rows of t: a group behind the other, pieces of 512 bytes
    const char *t0 = reinterpret_cast<const char *>(d.t) + row0 * d.tp * EB + (int64_t)((8 * h * EB / 16) * 512 + l32 * 16);
    const int64_t group = (int64_t)32 * d.tp * EB;
    auto steps = [&](int k, auto u_c) {
      constexpr int U = decltype(u_c)::value;
      if constexpr (!XF32) {
        ad_bf16x8_t a[U][TI], b[U][TJ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int j = 0; j < TJ; ++j) b[u][j] = adapter_b8(d, id * N + col[j], k + 16 * u + 8 * h);
#pragma unroll
          for (int i = 0; i < TI; ++i) a[u][i] = adapter_t8(t0 + i * group + (k / 8 + 2 * u) * 512, 512);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < TI; ++i) run(acc[i], a[u][i], b[u]);
      } else {
        float a[U][TI][8], b[U][TJ][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int j = 0; j < TJ; ++j) adapter_b8(d, id * N + col[j], k + 16 * u + 8 * h, b[u][j]);
#pragma unroll
          for (int i = 0; i < TI; ++i) adapter_t8(t0 + i * group + (k / 4 + 4 * u) * 512, 512, a[u][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Terms3 b3[TJ];
#pragma unroll
          for (int j = 0; j < TJ; ++j) b3[j] = terms3(b[u][j]);
#pragma unroll
          for (int i = 0; i < TI; ++i) run(acc[i], terms3(a[u][i]), b3);
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
  // several segments, or rows past the matrix: adapter after adapter
  constexpr int U = XF32 && TJ > 1 ? 2 : 4;  // steps of 16 rank values whose loads go together
  AdapterWalk<TI> step(d, M, row0, end, s);
  // a product to the adapter's rows of tile i alone: another's would be NaN where B is not finite
  auto add = [&](int i, uint32_t rows, const ad_f32x16_t (&own)[TJ]) {
    const uint32_t mine = rows >> (4 * h);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool in = mine >> (8 * (e >> 2) + (e & 3)) & 1;
#pragma unroll
      for (int j = 0; j < TJ; ++j) acc[i][j][e] += in ? own[j][e] : 0.f;
    }
  };
  if constexpr (TI > 1) {
    // a row tile's product over the whole rank: its rows are picked once
    while (step.next_adapter()) {
      int l = l32;
      asm volatile("" : "+v"(l));  // the row tiles' addresses are formed in each turn, not kept through the loop
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const bool in = step.has(i, step.who);
        const uint32_t rows = (uint32_t)__builtin_amdgcn_ballot_w64(in);
        if (!rows) continue;  // uniform
        ad_f32x16_t own[TJ] = {};
        for (int k = 0; k < d.tp; k += 16 * U) {
          std::conditional_t<XF32, Values8, ad_bf16x8_t> b[U][TJ], a[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (k + 16 * u >= d.tp) break;  // uniform
            const int ku = k + 16 * u + 8 * h;
            a[u] = adapter_t_row<XF32>(d, M, row0 + 32 * i + l, in, ku);
#pragma unroll
            for (int j = 0; j < TJ; ++j) b[u][j] = adapter_b<XF32>(d, (int64_t)step.adapter * N + col[j], ku);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (k + 16 * u >= d.tp) break;  // uniform
            std::conditional_t<XF32, Terms3, ad_bf16x8_t> bt[TJ];
#pragma unroll
            for (int j = 0; j < TJ; ++j) bt[j] = adapter_terms(b[u][j]);
            run(own, adapter_terms(a[u]), bt);
          }
        }
        add(i, rows, own);
      }
    }
    return;
  }
  bool more = step.next();
  while (more) {
    int who[U], n = 0;
    std::conditional_t<XF32, Values8, ad_bf16x8_t> b[U][TJ], a[U][TI];
    int l = l32;
    asm volatile("" : "+v"(l));  // the row tiles' addresses are formed in each turn, not kept through the loop
#pragma unroll
    for (int u = 0; u < U; ++u) {  // past the last step: no rows
      who[u] = step.who;
#pragma unroll
      for (int j = 0; j < TJ; ++j) b[u][j] = adapter_b<XF32>(d, (int64_t)step.adapter * N + col[j], step.k + 8 * h);
#pragma unroll
      for (int i = 0; i < TI; ++i)
        a[u][i] = adapter_t_row<XF32>(d, M, row0 + 32 * i + l, step.has(i, who[u]), step.k + 8 * h);
      if (more) {
        ++n;
        more = step.next();
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= n) break;  // uniform
      std::conditional_t<XF32, Terms3, ad_bf16x8_t> bt[TJ];
#pragma unroll
      for (int j = 0; j < TJ; ++j) bt[j] = adapter_terms(b[u][j]);
#pragma unroll
      for (int i = 0; i < TI; ++i) {
        const uint32_t rows = (uint32_t)__builtin_amdgcn_ballot_w64(step.has(i, who[u]));
        if (!rows) continue;  // uniform
        ad_f32x16_t own[TJ] = {};
        run(own, adapter_terms(a[u][i]), bt);
        add(i, rows, own);
      }
    }
  }
}

// The same for kernels of few rows: acc[i] += t B^T for rows row0 + 16 i .. and columns col0 .. of MT tiles of 16 x 16,
// which NW wavefronts share out: the steps of 32 rank values of the rows' segments, in turn. Segment by segment, not adapter
// by adapter as above: a wavefront's steps are few, and finding them costs instructions of every wavefront.
template <bool XF32, int MT, int NW>
__device__ __forceinline__ void adapter_add16(const AdapterParams &d, int64_t M, int64_t N, int64_t row0, int64_t col0,
                                              int wave, ad_f32x4_t (&acc)[MT]) {
  const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
  const int64_t last = row0 + 16 * MT < M ? row0 + 16 * MT : M, col = col0 + l16 < N ? col0 + l16 : N - 1;
  const int steps = (d.tp + 31) / 32;  // of a segment
  int at = wave;                       // the wavefront's step, counted from the next segment's first
  for (int64_t s0 = d.nseg > 64 ? adapter_segment(d, row0) : 0; s0 < d.nseg; s0 += 64) {
    // a segment a lane
    const int64_t s = s0 + lane;
    int64_t from = last, to = last;
    int id = -1;
    if (s < d.nseg) {
      from = adapter_row(d, M, s);
      to = adapter_row(d, M, s + 1);
      id = adapter_id(d, s);
    }
    const int lo = (int)((from > row0 ? from < last ? from : last : row0) - row0);
    const int hi = (int)((to < last ? to > row0 ? to : row0 : last) - row0);
    uint64_t mask = __builtin_amdgcn_ballot_w64(hi > lo && id >= 0);
    while (true) {
      for (; mask && at >= steps; at -= steps) mask &= mask - 1;
      if (!mask) break;
      const int of = __builtin_ctzll(mask), k = 32 * at + 8 * g;
      const int first = __builtin_amdgcn_readlane(lo, of), end = __builtin_amdgcn_readlane(hi, of);
      const auto b = adapter_b<XF32>(d, __builtin_amdgcn_readlane(id, of) * N + col, k);
      std::conditional_t<XF32, Values8, ad_bf16x8_t> a[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int r = 16 * i + l16;  // lanes past t's row: zeros
        a[i] = adapter_t_row<XF32>(d, M, row0 + r, k < d.tp && r >= first && r < end, k);
      }
      const auto bt = adapter_terms(b);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const auto at3 = adapter_terms(a[i]);
        ad_f32x4_t own = {};
        if constexpr (!XF32) {
          own = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at3, bt, own, 0, 0, 0);
        } else {
#pragma unroll
          for (int m = 2; m >= 0; --m)
#pragma unroll
            for (int x = 0; x <= m; ++x) own = __builtin_amdgcn_mfma_f32_16x16x32_bf16(at3.t[x], bt.t[m - x], own, 0, 0, 0);
        }
        // added to the segment's rows alone: another's would be NaN where B is not finite
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 16 * i + 4 * g + e;
          acc[i][e] += r >= first && r < end ? own[e] : 0.f;
        }
      }
      at += NW;
    }
    if (!(__builtin_amdgcn_ballot_w64(from < last) >> 63)) break;  // the next segments lie past the rows
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
