// mxfp4_gemm.hip -- linear layers on microscaled 4-bit weights for many rows:
// tiles of y on the matrix cores, operands through an LDS ring.
//
// A workgroup of WM x WN wavefronts computes a BM x BN tile, each wavefront TM x
// TN matrix tiles of 32 x 32 (x rows x weight rows). Gated: half of the tile's
// weight rows are the gate's, those of the same outputs in the same wavefront
// and lane, so that the activation and the product happen in registers.
//
// x's type decides the depth of a stage and the instruction:
//   packed   128 of k; v_mfma_scale_f32_32x32x64_f8f6f4, two a stage and tile
//   2 bytes   64 of k; v_mfma_f32_32x32x16_{bf16,f16}, four
//   f32       32 of k; x in three exact bf16 terms, two times three
// Weight codes become bf16 / f16 values in registers, after the LDS (one convert
// for two values): LDS and global traffic stay at half a byte a value.
//
// k order inside a stage: lane half h = lane / 32 holds, packed, block 2 h + s of
// the stage's four in sub-step s, so that its two scale bytes are adjacent; 2
// bytes, values 8 s .. + 7 of block h; f32, values 16 h + 8 s .. + 7 of the one
// block. Stages arrive by direct loads (buffer_load ... lds) NS - 1 ahead, with
// the 16-byte pieces of a row swizzled so that the reads below, 16 rows at a
// time, meet every bank once. One barrier a stage, before the last sub-step's
// products, as in the Q8_0 ring kernel.
//
// The weights are the matrix instruction's first operand: a lane then holds four
// consecutive outputs of one row of y, and the epilogue packs whole words.
#include <type_traits>

#include "mxfp4.hpp"

namespace lux3d {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));

// X: void (packed x), BF16, F16 or F32.
template <typename X, int WM_, int WN_, int TM_, int TN_, int NS_, bool GATED_>
struct MxTile {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, NS = NS_;
  static constexpr bool GATED = GATED_, PACKED = std::is_void_v<X>;
  static constexpr bool XF32 = std::is_same_v<X, F32>;
  static constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN;
  static constexpr int BNO = GATED ? BN / 2 : BN;          // outputs of the tile's rows
  static constexpr int WC = GATED ? TN * 16 : TN * 32;     // a wavefront's
  static constexpr int BK = PACKED ? 128 : XF32 ? 32 : 64, SUB = PACKED || XF32 ? 2 : 4;
  static constexpr int XROW = PACKED ? 64 : 128, WROW = BK / 2;  // bytes of a row's stage
  static constexpr int XL = BM * XROW, WL = BN * WROW, XS = PACKED ? BM * 4 : 0, WS = BN * 4;
  static constexpr int STAGE = XL + WL + XS + WS;
  static constexpr int XSEG = XL / 1024, WSEG = WL / 1024, SSEG = (XS + WS) / 256;  // direct loads of a stage
  static constexpr int SX = XSEG > NW ? XSEG / NW : 1, SW = WSEG > NW ? WSEG / NW : 1, SS = (SSEG + NW - 1) / NW;
  static constexpr int OPS = SX + SW + SS;                 // of each wavefront
  static constexpr int LDS = NS * STAGE;
  static_assert(XL % 1024 == 0 && WL % 1024 == 0 && BM % 64 == 0 && BNO % 64 == 0, "whole segments");
  static_assert((XSEG % NW == 0 || NW % XSEG == 0) && (WSEG % NW == 0 || NW % WSEG == 0), "even shares");
  static_assert(!GATED || TN % 2 == 0, "a gate tile beside every up tile");
  static_assert(NW * 32 * (WC * 4 + 16) + BN * 4 <= LDS, "the epilogue's rows fit");
  static_assert((NS - 2) * OPS < 64, "vmcnt");
};

template <typename X, int WM, int WN, int TM, int TN, int NS, bool GATED>
__global__ __launch_bounds__(64 * WM * WN, 1) void mx_gemm_kernel(MxLinearParams p, MxAct act, int tiles_m, int tiles_n) {
  using T = MxTile<X, WM, WN, TM, TN, NS, GATED>;
  constexpr int GM = 8;  // row tiles of a group
  __shared__ __align__(16) char ring[T::LDS];

  // XCD-contiguous ranges of tiles, groups of GM row tiles, as in q8_0_gemm_ring_kernel
  const int G = tiles_m * tiles_n, bid = (int)blockIdx.x;
  const int per = G / 8, rem = G % 8, xcd = bid % 8, pos = bid / 8;
  const int lid = (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + pos;
  const int group = lid / (GM * tiles_n), first_m = group * GM;
  const int gsize = tiles_m - first_m < GM ? tiles_m - first_m : GM;
  const int in_group = lid - group * GM * tiles_n;
  const int tm = first_m + in_group % gsize, tn = in_group / gsize;

  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, l32 = lane & 31;
  const int wm = wave / WN, wn = wave % WN;
  const int64_t m0 = (int64_t)tm * T::BM, c0 = (int64_t)tn * T::BNO;
  const int nblk = (int)(p.K / 32), nk = (int)((p.K + T::BK - 1) / T::BK);
  const int rest = nblk % (T::BK / 32);  // blocks of a last stage that is not whole

  // Direct loads. Rows past the matrix are clamped to its last: loaded, computed, never stored. A last stage that is not
  // whole reads on into the next row, or past the descriptor's end (nothing): zero_tail clears x and the scales there, and
  // any four bits are a finite weight. Descriptors span the tile's rows (of the scales, every group).
  constexpr int EB = T::PACKED ? 1 : T::XF32 ? 4 : 2;
  const int64_t xrow = T::PACKED ? p.K / 2 : p.ldx * EB, xk = T::PACKED ? p.K / 2 : p.K * EB, groups = (nblk + 3) / 4;
  const int64_t last_m = p.M - 1 - m0 < T::BM - 1 ? p.M - 1 - m0 : T::BM - 1;
  const int64_t ncols = p.N - c0 < T::BNO ? p.N - c0 : T::BNO;
  const char *xbase = reinterpret_cast<const char *>(T::PACKED ? (const void *)p.xq : p.x) + m0 * xrow;
  const i32x4_t xr = buffer_rsrc(xbase, last_m * xrow + xk);
  uint32_t xoff[T::SX], xto[T::SX], woff[T::SW], wto[T::SW];
  i32x4_t wsrc[T::SW];
#pragma unroll
  for (int i = 0; i < T::SX; ++i) {
    const int seg = (wave * T::SX + i) % T::XSEG;
    const int r = T::PACKED ? seg * 16 + (lane >> 2) : seg * 8 + (lane >> 3);
    const int c = T::PACKED ? (lane & 3) ^ ((r >> 2) & 3) : (lane & 7) ^ ((r >> 1) & 7);
    xoff[i] = (uint32_t)((r <= last_m ? r : last_m) * xrow + 16 * c);
    xto[i] = seg * 1024;
  }
#pragma unroll
  for (int i = 0; i < T::SW; ++i) {
    const int seg = (wave * T::SW + i) % T::WSEG;
    int r, c;  // row of the tile, 16-byte piece
    if constexpr (T::PACKED) {
      r = seg * 16 + (lane >> 2);
      c = (lane & 3) ^ ((r >> 2) & 3);
    } else if constexpr (T::XF32) {
      r = seg * 64 + lane;
      c = 0;
    } else {
      r = seg * 32 + (lane >> 1);
      c = (lane & 1) ^ ((r >> 3) & 1);
    }
    const bool second = GATED && __builtin_amdgcn_readfirstlane(r) >= T::BNO;  // a segment lies in one matrix
    wsrc[i] = buffer_rsrc((second ? p.w[1] : p.w[0]) + c0 * (p.K / 2), ncols * (p.K / 2));
    const int64_t col = second ? r - T::BNO : r;
    woff[i] = (uint32_t)((col < ncols ? col : ncols - 1) * (p.K / 2) + 16 * c);
    wto[i] = T::XL + seg * 1024;
  }
  // the scales: 64 rows' words a load
  i32x4_t ssrc[T::SS];
  uint32_t soff[T::SS], sto[T::SS], sstep[T::SS];
#pragma unroll
  for (int i = 0; i < T::SS; ++i) {
    const int seg = (wave * T::SS + i) % T::SSEG, r = seg * 64 + lane;
    sto[i] = T::XL + T::WL + seg * 256;
    const bool of_x = seg * 256 < T::XS;
    const int rw = of_x ? r : r - T::XS / 4;
    const bool second = GATED && !of_x && seg * 64 - T::XS / 4 >= T::BNO;
    const int64_t line = second ? rw - T::BNO : rw, rows = of_x ? p.M : p.N, have = of_x ? last_m + 1 : ncols;
    ssrc[i] = buffer_rsrc((of_x ? p.xs + m0 * 4 : (second ? p.ws[1] : p.ws[0]) + c0 * 4), ((groups - 1) * rows + have) * 4);
    soff[i] = (uint32_t)((line < have ? line : have - 1) * 4);
    sstep[i] = (uint32_t)(rows * 4);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)ring;
  auto issue = [&](int kt, int slot) {
    const uint32_t st = lds0 + slot * T::STAGE;
#pragma unroll
    for (int i = 0; i < T::SX; ++i) lds_load16(xr, xoff[i], (uint32_t)kt * T::XROW, __builtin_amdgcn_readfirstlane(st + xto[i]));
#pragma unroll
    for (int i = 0; i < T::SW; ++i) lds_load16(wsrc[i], woff[i], (uint32_t)kt * T::WROW, __builtin_amdgcn_readfirstlane(st + wto[i]));
#pragma unroll
    for (int i = 0; i < T::SS; ++i)
      lds_load4(ssrc[i], soff[i], __builtin_amdgcn_readfirstlane((uint32_t)(kt / (128 / T::BK)) * sstep[i]),
                __builtin_amdgcn_readfirstlane(st + sto[i]));
  };
  // A last stage that is not whole: zeros for x past its end, and for the scales of the blocks that are not there.
  auto zero_tail = [&](int slot) {
    char *st = ring + slot * T::STAGE;
    constexpr int CPR = T::XROW / 16, CPB = T::PACKED ? 1 : 4;  // pieces of a row, of a block
    for (int i = t; i < T::BM * CPR; i += 64 * T::NW) {
      const int r = i / CPR, c = i % CPR;
      if (c < rest * CPB) continue;
      const int at = T::PACKED ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7);
      *reinterpret_cast<uint4 *>(st + r * T::XROW + at * 16) = make_uint4(0, 0, 0, 0);
    }
    const int keep = (nblk - 1) % 4 + 1;  // scale bytes of the last group
    if (keep < 4)
      for (int i = t; i < (T::XS + T::WS) / 4; i += 64 * T::NW)
        reinterpret_cast<uint32_t *>(st + T::XL + T::WL)[i] &= (1u << (8 * keep)) - 1;
    lds_barrier();
  };

  // Fragments of a sub-step. Weight tile j lies in rows wrow(j) of the stage, x tile i in (wm TM + i) * 32.
  auto wrow = [&](int j) {
    if constexpr (GATED) return (j / (TN / 2)) * T::BNO + (wn * (TN / 2) + j % (TN / 2)) * 32;
    else return (wn * TN + j) * 32;
  };
  constexpr int XT = T::XF32 ? 3 : 1;  // terms of x
  struct XFrag { u32x4_t v[XT]; };
  XFrag xf[2][TM];
  u32x4_t wf[2][TN];
  u32x4_t wraw[TN];                 // plain: the stage's codes of a lane (f32: half of it used)
  uint32_t wsc[TN], xsc[TM];        // scales of the stage in use: packed two bytes, else one
  uint32_t wsn[TN], xsn[TM];        // and of the next
  auto read_stage = [&](int kt) {
    const char *st = ring + (kt % NS) * T::STAGE;
    const char *ws = st + T::XL + T::WL + T::XS;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int r = wrow(j) + l32;
      if constexpr (T::PACKED) {
        wsn[j] = *reinterpret_cast<const uint16_t *>(ws + r * 4 + 2 * h);
      } else if constexpr (T::XF32) {
        const uint2 u = *reinterpret_cast<const uint2 *>(st + T::XL + r * 16 + h * 8);
        wraw[j] = u32x4_t{u.x, u.y, 0, 0};
        wsn[j] = *reinterpret_cast<const uint8_t *>(ws + r * 4 + (kt & 3));
      } else {
        wraw[j] = *reinterpret_cast<const u32x4_t *>(st + T::XL + r * 32 + ((h ^ ((l32 >> 3) & 1)) << 4));
        wsn[j] = *reinterpret_cast<const uint8_t *>(ws + r * 4 + 2 * (kt & 1) + h);
      }
    }
    if constexpr (T::PACKED) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
        xsn[i] = *reinterpret_cast<const uint16_t *>(st + T::XL + T::WL + ((wm * TM + i) * 32 + l32) * 4 + 2 * h);
    }
  };
  auto read_frags = [&](int kt, int s, int buf) {
    const char *st = ring + (kt % NS) * T::STAGE;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if constexpr (T::PACKED) {
        const int r = wrow(j) + l32;
        wf[buf][j] = *reinterpret_cast<const u32x4_t *>(st + T::XL + r * 64 + (((2 * h + s) ^ ((l32 >> 2) & 3)) << 4));
      } else {
        wf[buf][j] = mx_values8<std::conditional_t<std::is_same_v<X, F16>, F16, BF16>>(wraw[j][s], wsn[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int r = (wm * TM + i) * 32 + l32;
      const char *row = st + r * T::XROW;
      if constexpr (T::PACKED) {
        xf[buf][i].v[0] = *reinterpret_cast<const u32x4_t *>(row + (((2 * h + s) ^ ((l32 >> 2) & 3)) << 4));
      } else if constexpr (T::XF32) {
        const int sw = (l32 >> 1) & 7;
        const float4 a = *reinterpret_cast<const float4 *>(row + (((4 * h + 2 * s) ^ sw) << 4));
        const float4 b = *reinterpret_cast<const float4 *>(row + (((4 * h + 2 * s + 1) ^ sw) << 4));
        const Split3 q[4] = {split3_bf16(a.x, a.y), split3_bf16(a.z, a.w), split3_bf16(b.x, b.y), split3_bf16(b.z, b.w)};
        xf[buf][i].v[0] = u32x4_t{q[0].t1, q[1].t1, q[2].t1, q[3].t1};
        xf[buf][i].v[XT / 2] = u32x4_t{q[0].t2, q[1].t2, q[2].t2, q[3].t2};
        xf[buf][i].v[XT - 1] = u32x4_t{q[0].t3, q[1].t3, q[2].t3, q[3].t3};
      } else {
        xf[buf][i].v[0] = *reinterpret_cast<const u32x4_t *>(row + (((4 * h + s) ^ ((l32 >> 1) & 7)) << 4));
      }
    }
  };
  f32x16_t acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[j][i] = f32x16_t{};
  auto products = [&](auto sub, int buf) {
    constexpr int S = decltype(sub)::value;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (T::PACKED) {
          const u32x4_t a = wf[buf][j], b = xf[buf][i].v[0];
          const i32x8_t av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
          const i32x8_t bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc[j][i], 4, 4, S, (int)wsc[j], S, (int)xsc[i]);
        } else if constexpr (std::is_same_v<X, F16>) {
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, wf[buf][j]),
                                                             __builtin_bit_cast(f16x8_t, xf[buf][i].v[0]), acc[j][i], 0, 0, 0);
        } else {
#pragma unroll
          for (int e = XT - 1; e >= 0; --e)  // smallest terms first
            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, wf[buf][j]),
                                                                __builtin_bit_cast(bf16x8_t, xf[buf][i].v[e]), acc[j][i], 0, 0, 0);
        }
      }
  };
  auto next_scales = [&]() {
#pragma unroll
    for (int j = 0; j < TN; ++j) wsc[j] = wsn[j];
    if constexpr (T::PACKED) {
#pragma unroll
      for (int i = 0; i < TM; ++i) xsc[i] = xsn[i];
    }
  };

  // Past the last stage the loop reloads it into slots that are not read for data again, so that the wait counts stay.
#pragma unroll
  for (int st = 0; st < NS - 1; ++st) issue(st < nk ? st : nk - 1, st);
  __builtin_amdgcn_s_waitcnt(waitcnt_vm((NS - 2) * T::OPS));  // stage 0 landed
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  if (rest && nk == 1) zero_tail(0);
  read_stage(0);
  read_frags(0, 0, 0);
  for (int kt = 0; kt < nk; ++kt) {
    next_scales();
    // the slot refilled here was last read in step kt - 1, before its barrier
    issue(kt + NS - 1 < nk ? kt + NS - 1 : nk - 1, (kt + NS - 1) % NS);
    __builtin_amdgcn_sched_barrier(0);
    read_frags(kt, 1, 1);
    products(std::integral_constant<int, 0>{}, 0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (T::SUB == 4) {
      read_frags(kt, 2, 0);
      products(std::integral_constant<int, 1>{}, 1);
      __builtin_amdgcn_sched_barrier(0);
      read_frags(kt, 3, 1);
      products(std::integral_constant<int, 2>{}, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    // stage kt + 1 landed (only those issued after it may be in flight), this wavefront's reads of stage kt are done; then
    // every one's
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((NS - 2) * T::OPS));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (rest && kt + 2 == nk) zero_tail((kt + 1) % NS);
    read_stage(kt + 1);
    read_frags(kt + 1, 0, 0);
    products(std::integral_constant<int, T::SUB - 1>{}, 1);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));  // the trailing reloads and reads
  __builtin_amdgcn_s_barrier();                     // every wavefront is done with the ring

  // Epilogue. Lane holds outputs 8 q + 4 h .. + 3 of weight tile j for row l32 of x tile i: bias, activation and product in
  // f32, one rounding, 32 rows of the wavefront's outputs at a time through LDS (rows padded by 16 bytes), whole 16-byte
  // pieces of y's rows out.
  float *const bias = reinterpret_cast<float *>(ring + T::LDS - T::BN * 4);
  for (int i = t; i < T::BN; i += 64 * T::NW) {
    const bool second = GATED && i >= T::BNO;
    const float *b = second ? p.bias[1] : p.bias[0];
    const int64_t col = c0 + (second ? i - T::BNO : i);
    bias[i] = b && col < p.N ? b[col] : 0.f;
  }
  lds_barrier();
  constexpr int TO = GATED ? TN / 2 : TN;  // output tiles of a wavefront
  auto write = [&](auto bytes) {
    constexpr int B = decltype(bytes)::value, ROW = T::WC * B + 16, CPR = T::WC * B / 16, EPC = 16 / B;
    char *const reg = ring + wave * 32 * ROW;
    const int64_t cw = c0 + wn * T::WC;
    const bool whole = (uintptr_t)p.y % 16 == 0 && p.ldy * B % 16 == 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TO; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 b0 = *reinterpret_cast<const float4 *>(bias + wrow(j) + 8 * q + 4 * h);
          float v[4] = {acc[j][i][4 * q] + b0.x, acc[j][i][4 * q + 1] + b0.y, acc[j][i][4 * q + 2] + b0.z, acc[j][i][4 * q + 3] + b0.w};
          if constexpr (GATED) {
            const float4 b1 = *reinterpret_cast<const float4 *>(bias + wrow(j + TO) + 8 * q + 4 * h);
            const float g[4] = {b1.x, b1.y, b1.z, b1.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= mx_activate(act, acc[j + TO][i][4 * q + e] + g[e]);
          }
          char *to = reg + l32 * ROW + (j * 32 + 8 * q + 4 * h) * B;
          if constexpr (B == 4) *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
          else if (p.y_dt == LUX3D_BF16) *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
          else *reinterpret_cast<uint2 *>(to) = make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
        }
      // the wavefront's own memory: its LDS operations keep their order, only the compiler has to know
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int it = 0; it < 32 * CPR / 64; ++it) {
        const int n = it * 64 + lane, r = n / CPR, part = n % CPR;
        const int64_t row = m0 + (wm * TM + i) * 32 + r, col = cw + part * EPC;
        if (row >= p.M || col >= p.N) continue;
        const uint4 v = *reinterpret_cast<const uint4 *>(reg + r * ROW + part * 16);
        char *dst = reinterpret_cast<char *>(p.y) + (row * p.ldy + col) * B;
        if (whole && col + EPC <= p.N) {
          *reinterpret_cast<uint4 *>(dst) = v;
        } else {
          const uint32_t w4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < EPC; ++e)
            if (col + e < p.N) {
              if constexpr (B == 4) reinterpret_cast<uint32_t *>(dst)[e] = w4[e];
              else reinterpret_cast<uint16_t *>(dst)[e] = (uint16_t)(w4[e >> 1] >> (16 * (e & 1)));
            }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (p.y_dt == LUX3D_F32) write(std::integral_constant<int, 4>{});
  else write(std::integral_constant<int, 2>{});
}

template <typename X, int WM, int WN, int TM, int TN, int NS, bool GATED>
hipError_t launch_tile(const MxLinearParams &p, hipStream_t s) {
  using T = MxTile<X, WM, WN, TM, TN, NS, GATED>;
  const int64_t tiles_m = (p.M + T::BM - 1) / T::BM, tiles_n = (p.N + T::BNO - 1) / T::BNO;
  if (tiles_m * tiles_n > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL((mx_gemm_kernel<X, WM, WN, TM, TN, NS, GATED>), dim3((unsigned)(tiles_m * tiles_n)), dim3(64 * T::NW), 0, s, p,
                     mx_act(p.act), (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <typename X, bool GATED>
hipError_t launch_gemm(const MxLinearParams &p, int tile, hipStream_t s) {
  if constexpr (std::is_void_v<X>) {
    if (tile == 256) return launch_tile<X, 2, 2, 4, 4, 4, GATED>(p, s);
  } else if constexpr (!std::is_same_v<X, F32>) {
    if (tile == 256) return launch_tile<X, 2, 4, 4, 2, 3, GATED>(p, s);
  }
  return launch_tile<X, 2, 2, 2, 2, std::is_void_v<X> ? 4 : 3, GATED>(p, s);
}

template <typename X>
hipError_t launch_gemm(const MxLinearParams &p, int tile, hipStream_t s) {
  return p.act >= 0 ? launch_gemm<X, true>(p, tile, s) : launch_gemm<X, false>(p, tile, s);
}

}  // namespace

// The kernel's descriptors span 256 rows of x and of the weights, and the scales of the whole matrix; its offsets have 32
// bits.
bool mx_gemm_fits(const MxLinearParams &p) {
  const int64_t lim = 0x7FFFFFFF, eb = p.x_dt == LUX3D_F32 ? 4 : 2;
  return 256 * (p.x ? p.ldx * eb + 64 : p.K / 2) <= lim && 256 * p.K <= lim && (p.K + 127) / 32 * p.N <= lim &&
         (p.K + 127) / 32 * p.M <= lim;
}

hipError_t launch_mx_gemm(const MxLinearParams &p, int tile, hipStream_t s) {
  if (!p.x) return launch_gemm<void>(p, tile, s);
  switch (p.x_dt) {
    case LUX3D_F32: return launch_gemm<F32>(p, tile, s);
    case LUX3D_BF16: return launch_gemm<BF16>(p, tile, s);
    case LUX3D_F16: return launch_gemm<F16>(p, tile, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lux3d
