// adapters.hip -- the first product of the low-rank adapters beside a Q8_0 linear: t = alpha x A^T for rows whose
// segment has an adapter (the second, t B^T, joins the GEMM's accumulators, adapters.hpp).
//
// What bounds it: x's bytes, or for few rows the latency of one load after the other. A workgroup takes 16 rows of one
// segment (past 256 segments: 16 rows, segment after segment) and 16 NT values of the rank; its wavefronts take 128-byte
// chunks of the rows in turn and their sums are added in wavefront order through LDS (v_mfma_f32_16x16x32_bf16, f32 sums;
// f32 x: v_mfma_f32_16x16x4_f32). A chunk goes through LDS, 8 lanes to a row: loaded as the matrix operand's lanes hold it,
// a row a lane, the cache serves 16 bytes a cycle.
// us, operand loads / through LDS: 4096 x 2048 rank 64 bf16 15.4 / 9.7, 3087 x 4096 rank 32 f32 26 / 18, 9001 x 1536 rank
// 12 bf16 11.0 / 8.1, 12 x 1536 rank 16 5.0 / 4.4 (50 MB of f32 x: 10.4 us at the copy rate). t is rounded once to x's
// type, as an activation between two linear layers is, and as the second product's operands are (error of y against 64
// bits 0.0019 of its norm in bf16, 0.0017 by y's own rounding alone).
#include "adapters.hpp"

namespace lux3d {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Tile `tile` of 16 rows within segments: its first row, the segment's end and adapter; id -1 past the last
// tile, too. Every lane of the wavefront calls it; lanes take one segment each.
struct AdapterTile {
  int64_t row, end;
  int id;
};
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterParams &d, int64_t rows, int64_t tile) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int64_t s0 = 0; s0 < d.nseg; s0 += 64) {
    const int64_t s = s0 + lane, a = adapter_row(d, rows, s), b = s < d.nseg ? adapter_row(d, rows, s + 1) : a;
    const int id = adapter_id(d, s < d.nseg ? s : d.nseg - 1);
    // tiles of the segment and of those up to it; below 2^31 both, as rows / 16
    const int n = b > a ? (int)((b - a + 15) / 16) : 0;
    int sum = n;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(sum, m, 64);
      if (lane >= m) sum += o;
    }
    // the first segment whose tiles reach past `tile`
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > tile);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int64_t first = before + __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(n, at);
      return {uniform(__shfl(a, at, 64) + (tile - first) * 16), uniform(__shfl(b, at, 64)),
              __builtin_amdgcn_readlane(id, at)};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return {0, 0, -1};
}

// TILES: workgroup x takes tile x of the segments' tiles. Else 16 rows from 16 x on, segment after segment: finding a tile
// takes every workgroup a round of loads for each 64 segments.
template <bool XF32, int NT, int NW, bool TILES>
__global__ __launch_bounds__(64 * NW) void adapter_down_kernel(AdapterDownParams p) {
  constexpr int EB = XF32 ? 4 : 2;
  constexpr int ROWS = 16 * (1 + NT), LD = ROWS / 8;  // rows of a chunk, x's and A's; its 1 KB loads
  __shared__ __align__(16) char lds[NW][ROWS * 128];
  const AdapterParams &d = p.ad;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = lane >> 4, l16 = lane & 15;
  const int j0 = (int)blockIdx.y * 16 * NT;
  if (p.bad && blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && wave == 0) {
    // segments whose id is neither -1 nor an adapter's; by the last workgroup, which seldom has a tile
    int bad = 0;
    for (int64_t s = lane; s < d.nseg; s += 64) bad += d.ids[s] < -1 || d.ids[s] >= d.n;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) bad += __shfl_xor(bad, m, 64);
    if (lane == 0) *p.bad = bad;
  }
  // rows w.row .. w.end - 1, at most 16 of them, of adapter w.id; uniform over the workgroup, as every branch on them
  auto rows_of = [&](const AdapterTile w) {
    const float alpha = d.alpha ? d.alpha[w.id] : 1.f;
    // load i: rows 8 i .. + 7, a lane 16 bytes: piece `piece` of row 8 i + lane / 8, kept in slot lane % 8. Rows past the
    // segment are clamped: loaded, computed, never stored; so are values past the rank.
    const int piece = (lane & 7) ^ (lane >> 3);
    const char *src[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r = 8 * i + (lane >> 3);
      if (i < 2) {
        const int64_t row = w.row + r < w.end ? w.row + r : w.end - 1;
        src[i] = reinterpret_cast<const char *>(p.x) + row * p.ldx * EB + piece * 16;
      } else {
        const int j = j0 + r - 16 < d.r ? j0 + r - 16 : d.r - 1;
        src[i] = reinterpret_cast<const char *>(d.a) + ((int64_t)w.id * d.r + j) * p.K * EB + piece * 16;
      }
    }
    f32x4_t acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = f32x4_t{};
    char *const my = lds[wave];
    uint4 v[LD];
    auto load = [&](int64_t at) {
#pragma unroll
      for (int i = 0; i < LD; ++i) v[i] = ld16<false>(src[i] + at);
    };
    auto store = [&]() {
#pragma unroll
      for (int i = 0; i < LD; ++i) *reinterpret_cast<uint4 *>(my + i * 1024 + lane * 16) = v[i];
      // the wavefront's own memory: its reads follow its writes in order, and only the compiler has to know
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    };
    // half q of the chunk: piece 4 q + g of the lane's row on both operands
    auto products = [&](int q) {
      const int off = l16 * 128 + (((4 * q + g) ^ (l16 & 7)) << 4);
      const uint4 x = *reinterpret_cast<const uint4 *>(my + off);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 a = *reinterpret_cast<const uint4 *>(my + (1 + n) * 2048 + off);
        if constexpr (!XF32) {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8_t, x), __builtin_bit_cast(ad_bf16x8_t, a),
                                                           acc[n], 0, 0, 0);
        } else {
          const f32x4_t xv = __builtin_bit_cast(f32x4_t, x), av = __builtin_bit_cast(f32x4_t, a);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[e], av[e], acc[n], 0, 0, 0);
        }
      }
    };
    const int64_t bytes = p.K * EB, nch = bytes / 128;  // chunks of 128 bytes a row
    if (wave < nch) load(wave * 128);
    for (int64_t c = wave; c < nch; c += NW) {
      store();
      if (c + NW < nch) load((c + NW) * 128);
      products(0);
      products(1);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if (bytes % 128 && wave == (int)(nch % NW)) {
      // the last 64 bytes; pieces 4 to 7 load what 0 to 3 do
      load(nch * 128 - (piece & 4) * 16);
      store();
      products(0);
    }
    __syncthreads();
    // lane holds rows 4 g + e, rank value lane % 16 of each tile
    float *const part = reinterpret_cast<float *>(lds);
    static_assert(NT * 1024 <= ROWS * 128, "partial sums fit");
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave * NT * 256 + n * 256 + e * 64 + lane] = acc[n][e];
    __syncthreads();
    for (int o = t; o < NT * 256; o += 64 * NW) {
      const int64_t r = w.row + 4 * ((o & 63) >> 4) + (o >> 6 & 3);
      const int j = j0 + (o >> 8) * 16 + (o & 15);
      if (r >= w.end || j >= d.tp) continue;
      float s = part[o];
#pragma unroll
      for (int k = 1; k < NW; ++k) s += part[k * NT * 256 + o];
      s = j < d.r ? s * alpha : 0.f;
      constexpr int E = 16 / EB;
      int next;
      char *to = adapter_t<EB>(d, p.M, r, j & -E, next);
      store1<std::conditional_t<XF32, F32, BF16>>(to, j & (E - 1), s);
    }
    if constexpr (!TILES) __syncthreads();  // the next segment's chunks
  };
  if constexpr (TILES) {
    const AdapterTile w = adapter_tile(d, p.M, blockIdx.x);
    if (w.id >= 0) rows_of(w);
  } else {
    const int64_t row0 = (int64_t)blockIdx.x * 16, last = row0 + 16 < p.M ? row0 + 16 : p.M;
    for (int64_t s0 = adapter_segment(d, row0); s0 < d.nseg; s0 += 64) {
      // a segment a lane
      const int64_t s = s0 + lane;
      int64_t from = last, to = last;
      int id = -1;
      if (s < d.nseg) {
        from = adapter_row(d, p.M, s);
        to = adapter_row(d, p.M, s + 1);
        id = adapter_id(d, s);
      }
      const int lo = (int)((from > row0 ? from < last ? from : last : row0) - row0);
      const int hi = (int)((to < last ? to > row0 ? to : row0 : last) - row0);
      for (uint64_t mask = __builtin_amdgcn_ballot_w64(hi > lo && id >= 0); mask; mask &= mask - 1) {
        const int of = __builtin_ctzll(mask);
        rows_of({row0 + __builtin_amdgcn_readlane(lo, of), row0 + __builtin_amdgcn_readlane(hi, of),
                 __builtin_amdgcn_readlane(id, of)});
      }
      if (!(__builtin_amdgcn_ballot_w64(from < last) >> 63)) break;  // the next segments lie past the rows
    }
  }
}

template <bool XF32, int NT, int NW>
hipError_t launch_down(const AdapterDownParams &p, hipStream_t s) {
  if (p.M > INT32_MAX) return hipErrorInvalidValue;
  const unsigned jt = (unsigned)((p.ad.tp + 16 * NT - 1) / (16 * NT));
  if (p.ad.nseg <= 256) {
    // at most one partly filled tile a segment
    int64_t tiles = p.M / 16 + p.ad.nseg;
    tiles = tiles < p.M ? tiles : p.M;
    hipLaunchKernelGGL((adapter_down_kernel<XF32, NT, NW, true>), dim3((unsigned)tiles, jt), dim3(64 * NW), 0, s, p);
  } else {
    hipLaunchKernelGGL((adapter_down_kernel<XF32, NT, NW, false>), dim3((unsigned)((p.M + 15) / 16), jt), dim3(64 * NW), 0, s, p);
  }
  return hipGetLastError();
}

template <bool XF32, int NT>
hipError_t launch_down(const AdapterDownParams &p, hipStream_t s) {
  // us of a call with 64 columns, with 4 / 8 wavefronts in this kernel: 1024 x 4096 f32 rank 8 31.9 / 27.7, 3087 x 2048 bf16
  // rank 8 18.8 / 17.7, 32768 x 1024 bf16 rank 32 37.4 / 43.0; over 24 sizes each, 8 take 0.94 of the time at 1024 rows, 0.97
  // at 3087, and 1.02 from 4096 rows on (0.98 to 1.07 up to 8192). The border stays above where the two meet: another number
  // of wavefronts is another order of t's sums.
  return p.M > 8192 ? launch_down<XF32, NT, 4>(p, s) : launch_down<XF32, NT, 8>(p, s);
}

}  // namespace

hipError_t launch_adapter_down(const AdapterDownParams &p, bool x_f32, hipStream_t s) {
  if (p.M <= 0) return hipSuccess;
  if (p.ad.tp <= 16) return x_f32 ? launch_down<true, 1>(p, s) : launch_down<false, 1>(p, s);
  if (p.ad.tp <= 32) return x_f32 ? launch_down<true, 2>(p, s) : launch_down<false, 2>(p, s);
  return x_f32 ? launch_down<true, 4>(p, s) : launch_down<false, 4>(p, s);
}

}  // namespace lux3d
