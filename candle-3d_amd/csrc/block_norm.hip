// block_norm.hip -- the norms on both sides of a transformer block's residual sum, one pass over the rows:
//   n     = Norm(h; post_w, post_b)                       the norm after the block
//   x_out = x + n * ls_gamma * gate[s]                    residual scale and the segment's gate
//   y     = Norm(x_out; pre_w, pre_b) * (scale[s] + 1) + shift[s]      the norm before the next one
// Norm is LayerNorm or RMSNorm (no mean). Every per-channel factor folds into four vectors of a segment,
//   x_out = x + a1 * (h - mean) * rstd + a0,   y = b1 * (x_out - mean') * rstd' + b0
// with a1 = post_w ls_gamma gate, a0 = post_b ls_gamma gate, b1 = pre_w (scale + 1), b0 = pre_b (scale + 1) + shift.
// All arithmetic is f32; x_out is rounded once to its type, and y's statistics and values are those of the rounded
// x_out. Reads x and h and writes x_out and y once: memory bounds it, 64000 x 1536 bf16 at 5.0 TB/s (156 us for 786 MB),
// 4098 x 2048 f16 at 3.9 TB/s (17.2 us), 1029 x 1024 f32 6.4 us.
//
// Statistics take two passes over the registers (the mean, then the centred squares). The row's values and sums are
// those of rows.hpp.
#include "rows.hpp"

namespace lux3d {

namespace {

// The folded vectors of segment seg at elements off .. off + 3 (a: the post norm's, b: the pre norm's).
struct Coef4 {
  float a1[4], a0[4], b1[4], b0[4];
};
__device__ __forceinline__ void piece4(const ModPiece &m, int64_t seg, int64_t off, float dflt, float (&v)[4]) {
  param4(m.p, m.dt, m.dt >= 0 ? seg * m.ld + off : 0, dflt, v);
  if (m.dt >= 0 && m.base_dt >= 0) {
    float b[4];
    param4(m.base, m.base_dt, off, 0.f, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = b[k] + v[k];
  }
}
__device__ __forceinline__ void fold_coef(float pw, float pb, float ls, float gate, float qw, float qb, float sc,
                                          float sh, float &a1, float &a0, float &b1, float &b0) {
  const float g = ls * gate, s1 = sc + 1.0f;
  a1 = pw * g;
  a0 = pb * g;
  b1 = qw * s1;
  b0 = __builtin_fmaf(qb, s1, sh);
}
__device__ __forceinline__ Coef4 coef4(const BlockNormParams &p, int64_t seg, int64_t off) {
  float pw[4], pb[4], ls[4], g[4], qw[4], qb[4], sc[4], sh[4];
  param4(p.post_w, p.post_w_dt, off, 1.f, pw);
  param4(p.post_b, p.post_b_dt, off, 0.f, pb);
  param4(p.gamma, p.gamma_dt, off, 1.f, ls);
  param4(p.pre_w, p.pre_w_dt, off, 1.f, qw);
  param4(p.pre_b, p.pre_b_dt, off, 0.f, qb);
  piece4(p.gate, seg, off, 1.f, g);
  piece4(p.scale, seg, off, 0.f, sc);
  piece4(p.shift, seg, off, 0.f, sh);
  Coef4 c;
#pragma unroll
  for (int k = 0; k < 4; ++k) fold_coef(pw[k], pb[k], ls[k], g[k], qw[k], qb[k], sc[k], sh[k], c.a1[k], c.a0[k], c.b1[k], c.b0[k]);
  return c;
}

// Raw 16-byte pieces of a chunk, loaded ahead and decoded where they are used.
template <typename T> struct RawChunk {
  uint4 q[T::bytes / 2];
};
template <typename T> __device__ __forceinline__ void decode_raw(const RawChunk<T> &r, float (&v)[8]) {
  if constexpr (T::bytes == 4) {
    const uint32_t w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(w[k]);
  } else {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t e = (w[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
      v[k] = T::code == LUX3D_BF16 ? bf16_bits_to_f32(e) : f16_bits_to_f32(e);
    }
  }
}

// MASK: the row ends inside the last chunks (d a multiple of 8): halves of a chunk past d read as zeros, stay zero and
// are not stored.
template <bool MASK> __device__ __forceinline__ bool inside(int64_t off, int64_t d) { return !MASK || off < d; }
template <typename T, bool MASK> __device__ __forceinline__ RawChunk<T> ld_raw_in(const char *row, ChunkAt a, int64_t d) {
  RawChunk<T> r{};
  if (inside<MASK>(a.o0, d)) r.q[0] = ld16(row + a.o0 * T::bytes);
  if constexpr (T::bytes == 4) {
    if (inside<MASK>(a.o1, d)) r.q[1] = ld16(row + a.o1 * 4);
  }
  return r;
}
template <typename T, bool MASK> __device__ __forceinline__ void st_row_in(char *row, ChunkAt a, int64_t d, const float (&v)[8]) {
  if constexpr (!MASK) {
    st_row<T>(row, a, v);
  } else if constexpr (T::bytes == 4) {
    if (a.o0 < d) st16(row + a.o0 * 4, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
    if (a.o1 < d) st16(row + a.o1 * 4, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
  } else {
    if (a.o0 < d) st_row<T>(row, a, v);
  }
}

// Normalises the row's registers in place: v = (v - mean) * rstd (RMS: v * rstd).
template <typename T, bool RMS, bool MASK, int NC, int TPR, int BLOCK>
__device__ __forceinline__ void normalise(float (&v)[NC][8], int t, int64_t d, float inv_d, float eps, float *red_a,
                                          float *red_b) {
  float mean = 0.f;
  if constexpr (!RMS) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[c][k];
    mean = row_total<TPR, BLOCK>(s, red_a) * inv_d;
  }
  float s2 = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const ChunkAt at = chunk_at<T, TPR>(c, t);
    const bool in0 = inside<MASK>(at.o0, d), in1 = T::bytes == 4 ? inside<MASK>(at.o1, d) : in0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (!RMS) v[c][k] = (k < 4 ? in0 : in1) ? v[c][k] - mean : 0.f;
      s2 += v[c][k] * v[c][k];
    }
  }
  const float rstd = 1.0f / sqrtf(row_total<TPR, BLOCK>(s2, red_b) * inv_d + eps);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[c][k] *= rstd;
}

// Long jobs: a workgroup owns a run of consecutive rows, one wavefront per row at a time. The folded vectors of the
// run's segment are formed once in LDS (4 * d floats) and read from there by every row; where the run crosses into
// the next segment they are formed again. The next row's x and h are loaded before this row's arithmetic.
template <typename T, int NC, bool RMS, bool MASK>
__global__ __launch_bounds__(kBlock) void block_norm_walk_kernel(BlockNormParams p, int64_t rows_per_wg) {
  constexpr int EB = T::bytes, WPB = kBlock / 64;
  extern __shared__ __align__(16) float lds_coef[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t d = p.d, w = NC * 512, begin = (int64_t)blockIdx.x * rows_per_wg;
  const int64_t end = begin + rows_per_wg < p.rows ? begin + rows_per_wg : p.rows;
  float *const a1 = lds_coef, *const a0 = a1 + w, *const b1 = a0 + w, *const b0 = b1 + w;
  const float inv_d = 1.0f / (float)d;
  const char *xs = reinterpret_cast<const char *>(p.x), *hs = reinterpret_cast<const char *>(p.h);
  char *xo = reinterpret_cast<char *>(p.x_out), *ys = reinterpret_cast<char *>(p.y);
  RawChunk<T> rx[NC], rh[NC];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      rx[c] = ld_raw_in<T, MASK>(xs + r * p.x_rs * EB, chunk_at<T, 64>(c, lane), d);
      rh[c] = ld_raw_in<T, MASK>(hs + r * p.h_rs * EB, chunk_at<T, 64>(c, lane), d);
    }
  };
  for (int64_t cur = begin; cur < end;) {
    const int64_t seg = segment_of(p.seg_off, p.nseg, p.rows_per_seg, cur);
    int64_t stop = end;
    if (seg + 1 < p.nseg) stop = p.seg_off ? p.seg_off[seg + 1] : (seg + 1) * p.rows_per_seg;
    stop = stop < end ? stop : end;
    stop = uniform(stop > cur ? stop : cur + 1);  // offsets that do not ascend: one row at a time
    int64_t row = cur + wave;
    if (row < stop) load(row);
    lds_barrier();  // the last segment's vectors are no longer read
    for (int64_t e = threadIdx.x * 4; e < w; e += kBlock * 4) {
      Coef4 c{};
      if (inside<MASK>(e, d)) c = coef4(p, seg, e);
      *reinterpret_cast<float4 *>(a1 + e) = make_float4(c.a1[0], c.a1[1], c.a1[2], c.a1[3]);
      *reinterpret_cast<float4 *>(a0 + e) = make_float4(c.a0[0], c.a0[1], c.a0[2], c.a0[3]);
      *reinterpret_cast<float4 *>(b1 + e) = make_float4(c.b1[0], c.b1[1], c.b1[2], c.b1[3]);
      *reinterpret_cast<float4 *>(b0 + e) = make_float4(c.b0[0], c.b0[1], c.b0[2], c.b0[3]);
    }
    lds_barrier();
    for (; row < stop; row += WPB) {
      float x[NC][8], v[NC][8];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        decode_raw<T>(rx[c], x[c]);
        decode_raw<T>(rh[c], v[c]);
      }
      if (row + WPB < stop) load(row + WPB);
      issue_fence();
      normalise<T, RMS, MASK, NC, 64, kBlock>(v, lane, d, inv_d, p.eps, nullptr, nullptr);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const ChunkAt at = chunk_at<T, 64>(c, lane);
        float m[8], a[8];
        lds_at(a1, at, m);
        lds_at(a0, at, a);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] = Chunk<T>::round_trip(x[c][k] + __builtin_fmaf(v[c][k], m[k], a[k]));
        st_row_in<T, MASK>(xo + row * p.xo_rs * EB, at, d, v[c]);
      }
      if (!ys) continue;
      normalise<T, RMS, MASK, NC, 64, kBlock>(v, lane, d, inv_d, p.eps, nullptr, nullptr);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const ChunkAt at = chunk_at<T, 64>(c, lane);
        float m[8], a[8];
        lds_at(b1, at, m);
        lds_at(b0, at, a);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] = __builtin_fmaf(v[c][k], m[k], a[k]);
        st_row_in<T, MASK>(ys + row * p.y_rs * EB, at, d, v[c]);
      }
    }
    cur = stop;
  }
}

// Short jobs: one row per workgroup of TPR threads, the vectors folded per row from the (cached) parameters.
template <typename T, int TPR, int NC, bool RMS, bool MASK>
__global__ __launch_bounds__(TPR) void block_norm_row_kernel(BlockNormParams p) {
  constexpr int EB = T::bytes;
  __shared__ float red[4][TPR / 64];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float inv_d = 1.0f / (float)p.d;
  const char *xr = reinterpret_cast<const char *>(p.x) + row * p.x_rs * EB;
  const char *hr = reinterpret_cast<const char *>(p.h) + row * p.h_rs * EB;
  float x[NC][8], v[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    decode_raw<T>(ld_raw_in<T, MASK>(hr, chunk_at<T, TPR>(c, t), p.d), v[c]);
    decode_raw<T>(ld_raw_in<T, MASK>(xr, chunk_at<T, TPR>(c, t), p.d), x[c]);
  }
  const int64_t seg = segment_of(p.seg_off, p.nseg, p.rows_per_seg, row);
  Coef4 q[NC][2];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const ChunkAt at = chunk_at<T, TPR>(c, t);
    q[c][0] = q[c][1] = Coef4{};
    if (inside<MASK>(at.o0, p.d)) q[c][0] = coef4(p, seg, at.o0);
    if (inside<MASK>(at.o1, p.d)) q[c][1] = coef4(p, seg, at.o1);
  }
  normalise<T, RMS, MASK, NC, TPR, TPR>(v, t, p.d, inv_d, p.eps, red[0], red[1]);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[c][k] = Chunk<T>::round_trip(x[c][k] + __builtin_fmaf(v[c][k], q[c][k >> 2].a1[k & 3], q[c][k >> 2].a0[k & 3]));
    st_row_in<T, MASK>(reinterpret_cast<char *>(p.x_out) + row * p.xo_rs * EB, chunk_at<T, TPR>(c, t), p.d, v[c]);
  }
  if (!p.y) return;
  normalise<T, RMS, MASK, NC, TPR, TPR>(v, t, p.d, inv_d, p.eps, red[2], red[3]);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[c][k] = __builtin_fmaf(v[c][k], q[c][k >> 2].b1[k & 3], q[c][k >> 2].b0[k & 3]);
    st_row_in<T, MASK>(reinterpret_cast<char *>(p.y) + row * p.y_rs * EB, chunk_at<T, TPR>(c, t), p.d, v[c]);
  }
}

// Any width and alignment: one 256-thread workgroup per row, several passes over it (all but the first from L2).
template <typename T, bool RMS>
__global__ __launch_bounds__(kBlock) void block_norm_any_kernel(BlockNormParams p) {
  __shared__ float red[4][kBlock / 64];
  const int64_t row = blockIdx.x, d = p.d;
  const int64_t seg = segment_of(p.seg_off, p.nseg, p.rows_per_seg, row);
  const float inv_d = 1.0f / (float)d;
  auto piece = [&](const ModPiece &m, int64_t c, float dflt) -> float {
    if (m.dt < 0) return dflt;
    const float v = param1(m.p, m.dt, seg * m.ld + c, dflt);
    return m.base_dt >= 0 ? param1(m.base, m.base_dt, c, 0.f) + v : v;
  };
  auto coef = [&](int64_t c, float &a1, float &a0, float &b1, float &b0) {
    fold_coef(param1(p.post_w, p.post_w_dt, c, 1.f), param1(p.post_b, p.post_b_dt, c, 0.f),
              param1(p.gamma, p.gamma_dt, c, 1.f), piece(p.gate, c, 1.f), param1(p.pre_w, p.pre_w_dt, c, 1.f),
              param1(p.pre_b, p.pre_b_dt, c, 0.f), piece(p.scale, c, 0.f), piece(p.shift, c, 0.f), a1, a0, b1, b0);
  };
  // mean and rstd of the values f(c)
  auto stats = [&](auto f, float *ra, float *rb, float &mean, float &rstd) {
    mean = 0.f;
    if constexpr (!RMS) {
      float s = 0.f;
      for (int64_t c = threadIdx.x; c < d; c += kBlock) s += f(c);
      mean = row_total<kBlock>(s, ra) * inv_d;
    }
    float s2 = 0.f;
    for (int64_t c = threadIdx.x; c < d; c += kBlock) {
      const float dv = f(c) - mean;
      s2 += dv * dv;
    }
    rstd = 1.0f / sqrtf(row_total<kBlock>(s2, rb) * inv_d + p.eps);
  };
  float mean, rstd, mean2 = 0.f, rstd2 = 0.f;
  stats([&](int64_t c) { return load1<T>(p.h, row * p.h_rs + c); }, red[0], red[1], mean, rstd);
  auto xnew = [&](int64_t c, float a1, float a0) {
    const float n = (load1<T>(p.h, row * p.h_rs + c) - mean) * rstd;
    return Chunk<T>::round_trip(load1<T>(p.x, row * p.x_rs + c) + __builtin_fmaf(n, a1, a0));
  };
  if (p.y)
    stats(
        [&](int64_t c) {
          float a1, a0, b1, b0;
          coef(c, a1, a0, b1, b0);
          return xnew(c, a1, a0);
        },
        red[2], red[3], mean2, rstd2);
  for (int64_t c = threadIdx.x; c < d; c += kBlock) {
    float a1, a0, b1, b0;
    coef(c, a1, a0, b1, b0);
    const float xv = xnew(c, a1, a0);
    store1<T>(p.x_out, row * p.xo_rs + c, xv);
    if (p.y) store1<T>(p.y, row * p.y_rs + c, __builtin_fmaf((xv - mean2) * rstd2, b1, b0));
  }
}

template <typename T, bool RMS>
hipError_t launch_block_norm_t(const BlockNormParams &p, bool vec, hipStream_t s) {
  if (p.rows > INT32_MAX) return hipErrorInvalidValue;
  const int64_t chunks = p.d / 8;
  if (vec && p.rows >= 2048 && chunks <= 256) {
    // Two or three workgroups a CU walk the rows, four at a time: three where they take no more turns in all. us with 2 / 3
    // of them (inputs warm): RMS 3000 x 1536 bf16 11.8 / 8.9, LayerNorm 4098 x 2048 f16 17.2 / 15.5, 12000 x 1024 f32 36.9 /
    // 35.6, 64000 x 1536 bf16 159 / 155, but 2048 x 2048 f32 14.9 / 16.6, 8192 x 1024 bf16 13.5 / 13.9, 32768 x 2048 f16 104 /
    // 110. Rows that end inside a chunk gain less (24000 x 1000 bf16 41.6 / 43.8), f32 rows above 1024 from 12000 rows on only
    // (78.6 / 74.8; 4098 x 2048 26.5 / 29.6). A workgroup a row takes 1.2 to 1.7 times as long from 3000 rows of 2 bytes on,
    // and 0.6 to 0.95 of it at 1029.
    const int nc = (int)((chunks + 63) / 64);
    const int64_t cus = cu_count(s);
    auto turns = [&](int64_t wgs) { return wgs * (((p.rows + wgs * cus - 1) / (wgs * cus) + 3) / 4); };
    const bool three = turns(3) <= turns(2) && (T::bytes == 2 || nc <= 2 || p.rows >= 12000);
    const int64_t wgs = (three ? 3 : 2) * cus, per = (p.rows + wgs - 1) / wgs;
    const dim3 grid((unsigned)((p.rows + per - 1) / per));
    const size_t lds = (size_t)nc * 512 * 16;
#define LUX3D_WALK(NC_)                                                                                             \
  if (nc == NC_) {                                                                                                  \
    if (chunks % 64) hipLaunchKernelGGL((block_norm_walk_kernel<T, NC_, RMS, true>), grid, dim3(kBlock), lds, s, p, per); \
    else hipLaunchKernelGGL((block_norm_walk_kernel<T, NC_, RMS, false>), grid, dim3(kBlock), lds, s, p, per);      \
    return hipGetLastError();                                                                                       \
  }
    LUX3D_WALK(1) LUX3D_WALK(2) LUX3D_WALK(3) LUX3D_WALK(4)
#undef LUX3D_WALK
  }
  const dim3 grid((unsigned)p.rows);
#define LUX3D_ROW(TPR_, NC_)                                                                                      \
  if (vec && chunks <= TPR_ * NC_) {                                                                              \
    if (chunks < TPR_ * NC_) hipLaunchKernelGGL((block_norm_row_kernel<T, TPR_, NC_, RMS, true>), grid, dim3(TPR_), 0, s, p); \
    else hipLaunchKernelGGL((block_norm_row_kernel<T, TPR_, NC_, RMS, false>), grid, dim3(TPR_), 0, s, p);        \
    return hipGetLastError();                                                                                     \
  }
  LUX3D_ROW(64, 1) LUX3D_ROW(128, 1) LUX3D_ROW(192, 1) LUX3D_ROW(256, 1) LUX3D_ROW(256, 2) LUX3D_ROW(256, 4)
#undef LUX3D_ROW
  hipLaunchKernelGGL((block_norm_any_kernel<T, RMS>), grid, dim3(kBlock), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_norm(int dt, const BlockNormParams &p, bool vec, hipStream_t s) {
  if (p.rows <= 0) return hipSuccess;
  switch (dt) {
    case LUX3D_F32: return p.rms ? launch_block_norm_t<F32, true>(p, vec, s) : launch_block_norm_t<F32, false>(p, vec, s);
    case LUX3D_BF16: return p.rms ? launch_block_norm_t<BF16, true>(p, vec, s) : launch_block_norm_t<BF16, false>(p, vec, s);
    case LUX3D_F16: return p.rms ? launch_block_norm_t<F16, true>(p, vec, s) : launch_block_norm_t<F16, false>(p, vec, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lux3d
