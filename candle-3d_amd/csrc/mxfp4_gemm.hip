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
// block. Stages arrive by direct loads (buffer_load ... lds) ahead of their use,
// with the 16-byte pieces of a row swizzled so that the reads below, 16 rows at a
// time, meet every bank once. One barrier a stage.
//
// A sub-step's fragments are read during the products of the one before.
//
// KG: where tiles are few, KG groups of a workgroup's wavefronts take every KG th
// stage through rings of their own and add their sums in group order at the end:
// a lone tile's time is its chain of stages, not its bytes or products.
//
// PERSIST: as many workgroups as CUs, each with the next of its tiles. The first
// stages of the next tile are loaded during the last products of this one, and
// its stores drain during the next tile's products.
//
// 16384 x 8192 -> 8192 of packed x 539 us (4.08 PFLOP/s), of bf16 1519 (1.45): the
// chip's power bounds both. With zeros for data the first takes 395 (2.35 GHz
// instead of 1.58), 4096 x 8192 -> 2048 of bf16 81 instead of 114. y's stores, in
// bursts at the tiles' ends, take 30 of 170 us of 16384 x 2048 -> 8192 packed.
//
// The weights are the matrix instruction's first operand: a lane then holds four
// consecutive outputs of one row of y, and the epilogue packs whole words.
#include <utility>

#include "mxfp4_rows.hpp"

namespace lux3d {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <typename F, int... I>
__device__ __forceinline__ void for_each_slot(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// X: void (packed x), BF16, F16 or F32.
template <typename X, int WM_, int WN_, int TM_, int TN_, int NS_, int KG_, bool PERSIST_, bool GATED_>
struct MxTile {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, NS = NS_, KG = KG_;
  static constexpr bool PERSIST = PERSIST_, GATED = GATED_, PACKED = std::is_void_v<X>;
  static constexpr bool XF32 = std::is_same_v<X, F32>;
  static constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN;
  static constexpr int NG = GATED ? 2 : 1, BNO = BN / NG;        // matrices; outputs of the tile's rows
  static constexpr int TO = TN / NG, WC = 32 * TO;               // output tiles and outputs of a wavefront
  static constexpr int BK = PACKED ? 128 : XF32 ? 32 : 64, SUB = PACKED || XF32 ? 2 : 4;
  static constexpr int XROW = PACKED ? 64 : 128, WROW = BK / 2;  // bytes of a row's stage
  static constexpr int XL = BM * XROW, WL = BN * WROW, XS = PACKED ? BM * 4 : 0, WS = BN * 4;
  static constexpr int STAGE = XL + WL + XS + WS;
  static constexpr int XSEG = XL / 1024, WSEG = WL / 1024, SSEG = (XS + WS) / 256, BSEG = BN / 64;  // direct loads
  static constexpr int SX = XSEG > NW ? XSEG / NW : 1, SW = WSEG > NW ? WSEG / NW : 1, SS = (SSEG + NW - 1) / NW;
  static constexpr int SB = (BSEG + NW - 1) / NW;
  static constexpr int OPS = SX + SW + SS;                       // of each wavefront and stage
  static constexpr int OROW = 128 + 16, OUT = NW * 32 * OROW;    // the epilogue's rows: 128 bytes of 32 rows a wavefront
  static constexpr int BIAS = NS * STAGE, OUT_AT = PERSIST ? BIAS + 2 * BN * 4 : 0;
  static constexpr int RING = PERSIST ? OUT_AT + OUT : BIAS + BN * 4;  // of a group of wavefronts
  static constexpr int PART = TM * TN * 16 * 64 * 4;             // a wavefront's sums
  static constexpr int LDS = KG * RING;
  static_assert(XL % 1024 == 0 && WL % 1024 == 0 && BM % 64 == 0 && BNO % 64 == 0, "whole segments");
  static_assert((XSEG % NW == 0 || NW % XSEG == 0) && (WSEG % NW == 0 || NW % WSEG == 0), "even shares");
  static_assert(!GATED || TN % 2 == 0, "a gate tile beside every up tile");
  static_assert(mx_rows_lds<GATED, 1, 2, NW * KG> <= LDS, "a few rows' sums fit");
  static_assert(OUT_AT + OUT <= (PERSIST ? RING : BIAS) && LDS <= 160 * 1024, "the epilogue's rows fit");
  static_assert(KG == 1 || (!PERSIST && NW * PART <= RING), "a group's sums fit its ring");
  static_assert(NS >= 3 && (NS - 2) * OPS < 63, "stages");
};

template <typename X, int WM, int WN, int TM, int TN, int NS, int KG, bool PERSIST, bool GATED>
__global__ __launch_bounds__(64 * WM * WN * KG, 2) void mx_gemm_kernel(MxLinearParams p, MxAct act, int tiles_m, int tiles_n) {
  using T = MxTile<X, WM, WN, TM, TN, NS, KG, PERSIST, GATED>;
  constexpr int GM = 8;  // row tiles of a group
  __shared__ __align__(16) char lds[T::LDS];

  // group kg of the wavefronts takes every KG th stage through a ring of its own
  const int kg = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * T::NW)) : 0;
  const int t = KG > 1 ? threadIdx.x - kg * 64 * T::NW : threadIdx.x;
  const int lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, l32 = lane & 31;
  char *const ring = lds + kg * T::RING;
  const int wm = wave / WN, wn = wave % WN;
  const int nblk = (int)(p.K / 32), all = (int)((p.K + T::BK - 1) / T::BK), nk = (all + KG - 1) / KG;  // a group's stages
  const int rest = nblk % (T::BK / 32);           // blocks of a last stage that is not whole
  const bool tail = rest != 0 || all % KG != 0;   // the groups' last stages need zeros

  // Tiles: each XCD (workgroup id % 8) takes a contiguous range, in groups of GM row tiles, as in q8_0_gemm_ring_kernel; its
  // workgroups take the range's tiles in turn.
  const int G = tiles_m * tiles_n, xcd = (int)blockIdx.x % 8, per = G / 8, rem = G % 8;
  const int first = xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per, end = first + per + (xcd < rem ? 1 : 0);
  const int step = ((int)gridDim.x - xcd + 7) / 8;  // PERSIST
  int lid = first + (int)blockIdx.x / 8;
  // Rows past the last tile (2 x 2049 tokens): in shares of 32 outputs by workgroups behind the tiles', which run beside them
  // on a CU, PERSIST by the tiles' own at their end. (In a launch of their own:
  // f32 1029 x 1024 -> 4096 31.8 us against 28.4, gated f32 58.9 against 53.5.)
  auto few_rows = [&](int share) {
    mx_rows_tile<X, T::PACKED, GATED, 1, 2, T::NW * KG>(p, act, p.M, p.M + p.rest, (int64_t)share * 32, reinterpret_cast<float *>(lds));
  };
  if (!PERSIST && (int)blockIdx.x >= G) {
    few_rows((int)blockIdx.x - G);
    return;
  }
  if (lid >= end) return;
  int64_t m0 = 0, c0 = 0;  // of the tile that is computed
  auto place = [&](int id, int64_t &m, int64_t &c) {
    const int group = id / (GM * tiles_n), first_m = group * GM;
    const int gsize = tiles_m - first_m < GM ? tiles_m - first_m : GM;
    const int in_group = id - group * GM * tiles_n;
    m = (int64_t)(first_m + in_group % gsize) * T::BM;
    c = (int64_t)(in_group / gsize) * T::BNO;
  };

  // Direct loads. A lane's offsets are the same for every tile; the descriptors span the tile's rows (of the scales, every
  // group). Rows past the matrix lie past the descriptor: they are not read, and what the LDS holds there reaches only
  // outputs that are not stored. A last stage that is not whole reads on into the next row: zero_tail clears x and the
  // scales there, and any four bits are a finite weight.
  constexpr int EB = T::PACKED ? 1 : T::XF32 ? 4 : 2;
  const int64_t xrow = T::PACKED ? p.K / 2 : p.ldx * EB, xk = T::PACKED ? p.K / 2 : p.K * EB, groups = (nblk + 3) / 4;
  const char *const xbase = reinterpret_cast<const char *>(T::PACKED ? (const void *)p.xq : p.x);
  uint32_t xoff[T::SX], xto[T::SX], woff[T::SW], wto[T::SW], soff[T::SS], sto[T::SS];
  bool wgate[T::SW], sgate[T::SS], sx[T::SS];  // uniform: the gate's weights, the gate's scales, x's scales
#pragma unroll
  for (int i = 0; i < T::SX; ++i) {
    const int seg = (wave * T::SX + i) % T::XSEG;
    const int r = T::PACKED ? seg * 16 + (lane >> 2) : seg * 8 + (lane >> 3);
    const int c = T::PACKED ? (lane & 3) ^ ((r >> 2) & 3) : (lane & 7) ^ ((r >> 1) & 7);
    xoff[i] = (uint32_t)(r * xrow + 16 * c);
    xto[i] = seg * 1024;
  }
#pragma unroll
  for (int i = 0; i < T::SW; ++i) {
    const int seg = (wave * T::SW + i) % T::WSEG;  // lies in one matrix
    int r, c;                                      // row of the tile, 16-byte piece
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
    wgate[i] = GATED && seg >= T::WSEG / 2;
    woff[i] = (uint32_t)((r - (wgate[i] ? T::BNO : 0)) * (p.K / 2) + 16 * c);
    wto[i] = T::XL + seg * 1024;
  }
#pragma unroll
  for (int i = 0; i < T::SS; ++i) {  // 64 rows' words a load
    const int seg = (wave * T::SS + i) % T::SSEG, r = seg * 64 - T::XS / 4;
    sx[i] = r < 0;
    sgate[i] = GATED && r >= T::BNO;
    soff[i] = (uint32_t)((sx[i] ? seg * 64 : sgate[i] ? r - T::BNO : r) + lane) * 4;
    sto[i] = T::XL + T::WL + seg * 256;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + kg * T::RING;
  // the tile that is loaded: its descriptors, and the stage that comes next
  i32x4_t xr, wr[T::SW], sr[T::SS];  // one of each load, where it may be of either matrix
  int load_lid = lid, load_kt = kg, bias_buf = 0;
#pragma unroll
  for (int i = 0; i < T::SX; ++i) xto[i] = __builtin_amdgcn_readfirstlane(lds0 + xto[i]);
#pragma unroll
  for (int i = 0; i < T::SW; ++i) wto[i] = __builtin_amdgcn_readfirstlane(lds0 + wto[i]);
#pragma unroll
  for (int i = 0; i < T::SS; ++i) sto[i] = __builtin_amdgcn_readfirstlane(lds0 + sto[i]);
  auto load_tile = [&]() {
    int64_t m, c;
    place(load_lid, m, c);
    const int64_t rows = p.M - m < T::BM ? p.M - m : T::BM, cols = p.N - c < T::BNO ? p.N - c : T::BNO;
    xr = buffer_rsrc(xbase + m * xrow, (rows - 1) * xrow + xk);
#pragma unroll
    for (int i = 0; i < T::SW; ++i) wr[i] = buffer_rsrc((wgate[i] ? p.w[1] : p.w[0]) + c * (p.K / 2), cols * (p.K / 2));
#pragma unroll
    for (int i = 0; i < T::SS; ++i)
      sr[i] = buffer_rsrc(sx[i] ? p.xs + m * 4 : (sgate[i] ? p.ws[1] : p.ws[0]) + c * 4,
                          ((groups - 1) * (sx[i] ? p.xs_rows : p.N) + (sx[i] ? rows : cols)) * 4);
    // biases, ahead of the tile's first stage (columns past the matrix: not read, not used; no bias: the zeros stay)
#pragma unroll
    for (int i = 0; i < T::SB; ++i) {
      const int seg = (wave * T::SB + i) % T::BSEG;
      const bool gate = GATED && seg >= T::BSEG / 2;
      const float *b = gate ? p.bias[1] : p.bias[0];
      if (!b || kg > 0) continue;  // uniform
      const i32x4_t br = buffer_rsrc(b + c, cols * 4);
      lds_load4(br, (uint32_t)((seg - (gate ? T::BSEG / 2 : 0)) * 64 + lane) * 4, 0,
                __builtin_amdgcn_readfirstlane(lds0 + T::BIAS + bias_buf * T::BN * 4 + seg * 256));
    }
    if constexpr (PERSIST) bias_buf ^= 1;
  };
  auto issue = [&](int n, int to) {  // the n-th of OPS loads of the next stage, into slot `to`
    if (n < T::SX) {
      lds_load16(xr, xoff[n], (uint32_t)load_kt * T::XROW, __builtin_amdgcn_readfirstlane(xto[n] + to * T::STAGE));
    } else if (n < T::SX + T::SW) {
      const int i = n - T::SX;
      lds_load16(wr[i], woff[i], (uint32_t)load_kt * T::WROW, __builtin_amdgcn_readfirstlane(wto[i] + to * T::STAGE));
    } else {
      const int i = n - T::SX - T::SW;
      const uint32_t rows4 = (uint32_t)((sx[i] ? p.xs_rows : p.N) * 4);
      lds_load4(sr[i], soff[i], __builtin_amdgcn_readfirstlane((uint32_t)(load_kt / (128 / T::BK)) * rows4),
                __builtin_amdgcn_readfirstlane(sto[i] + to * T::STAGE));
    }
  };
  // Behind the last load of a stage. Past the last stage of the last tile that stage is loaded again, into slots that are
  // not read for data any more, so that the wait counts stay.
  auto advance = [&]() {
    if (load_kt + KG < all) {
      load_kt += KG;
    } else if (PERSIST && load_lid + step < end) {
      load_lid += step;
      load_kt = 0;
      load_tile();
    }
  };
  // A group's last stage where it is not whole, or not there (the stage before was loaded again): zeros for x past its end,
  // and for the scales of the blocks that are not there.
  auto zero_tail = [&](int slot) {
    char *st = ring + slot * T::STAGE;
    constexpr int CPR = T::XROW / 16, CPB = T::PACKED ? 1 : T::XF32 ? 8 : 4;  // pieces of a row, of a block
    const int last = (nk - 1) * KG + kg, have = last >= all ? 0 : last + 1 == all && rest ? rest : T::BK / 32;
    for (int i = t; i < T::BM * CPR; i += 64 * T::NW) {
      const int r = i / CPR, c = i % CPR;
      if (c < have * CPB) continue;
      const int at = T::PACKED ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7);
      *reinterpret_cast<uint4 *>(st + r * T::XROW + at * 16) = make_uint4(0, 0, 0, 0);
    }
    const int keep = last >= all ? 0 : (nblk - 1) % 4 + 1;  // scale bytes of the last group of blocks
    if (last + 1 >= all && keep < 4)
      for (int i = t; i < (T::XS + T::WS) / 4; i += 64 * T::NW)
        reinterpret_cast<uint32_t *>(st + T::XL + T::WL)[i] &= (1u << (8 * keep)) - 1;
    lds_barrier();
  };

  // Fragments. Weight tile j lies in rows (j / TO) BNO + (wn TO + j % TO) 32 of the stage, x tile i in (wm TM + i) 32. A lane's
  // place in a stage: of x for each 16-byte piece that it reads, of the weights, of the scales
  constexpr int XPC = T::PACKED ? 2 : 4;             // pieces of a lane
  int xat[XPC], wat[2], wsat, xsat = 0;
#pragma unroll
  for (int c = 0; c < XPC; ++c)
    xat[c] = (wm * TM * 32 + l32) * T::XROW + (T::PACKED ? ((2 * h + c) ^ ((l32 >> 2) & 3)) << 4 : ((4 * h + c) ^ ((l32 >> 1) & 7)) << 4);
  const int w0 = wn * T::TO * 32 + l32;              // row of the first weight tile; tile j: wtile(j) further
  auto wtile = [](int j) { return (j / T::TO) * T::BNO + j % T::TO * 32; };
#pragma unroll
  for (int c = 0; c < 2; ++c)
    wat[c] = T::XL + w0 * T::WROW + (T::PACKED ? ((2 * h + c) ^ ((l32 >> 2) & 3)) << 4 : T::XF32 ? h * 8 : (h ^ ((l32 >> 3) & 1)) << 4);
  wsat = T::XL + T::WL + T::XS + w0 * 4 + (T::XF32 ? 0 : 2 * h);
  if constexpr (T::PACKED) xsat = T::XL + T::WL + (wm * TM * 32 + l32) * 4 + 2 * h;
  else if constexpr (!T::XF32) wsat -= h;            // one byte: h, and 2 more in every second stage
  constexpr int XP = T::XF32 ? 2 : 1;                // 16-byte pieces of x's fragment
  struct Frag { u32x4_t v[XP]; };
  Frag xf[2][TM];
  u32x4_t wf[2][TN];                                 // plain: converted
  u32x4_t wraw[TN];                                  // plain: the stage's codes of a lane (f32: half of it used)
  uint32_t wsc[2][TN], xsc[2][TM];                   // scales: packed two bytes, else one
  // the n-th of NRS reads of a stage's scales, plain with its weights, into buffer b
  constexpr int NRS = T::PACKED ? TN + TM : TN;
  auto read_stage = [&](int slot, int kt, int n, int b) {
    const char *st = ring + slot * T::STAGE;
    if (n < TN) {
      if constexpr (T::PACKED) {
        wsc[b][n] = *reinterpret_cast<const uint16_t *>(st + wsat + wtile(n) * 4);
      } else if constexpr (T::XF32) {
        const uint2 u = *reinterpret_cast<const uint2 *>(st + wat[0] + wtile(n) * T::WROW);
        wraw[n] = u32x4_t{u.x, u.y, 0, 0};
        wsc[b][n] = *reinterpret_cast<const uint8_t *>(st + wsat + wtile(n) * 4 + (kt & 3));
      } else {
        wraw[n] = *reinterpret_cast<const u32x4_t *>(st + wat[0] + wtile(n) * T::WROW);
        wsc[b][n] = *reinterpret_cast<const uint8_t *>(st + wsat + wtile(n) * 4 + 2 * (kt & 1));
      }
    } else if constexpr (T::PACKED) {
      xsc[b][n - TN] = *reinterpret_cast<const uint16_t *>(st + xsat + (n - TN) * 128);
    }
  };
  typedef std::conditional_t<std::is_same_v<X, F16>, F16, BF16> WT;  // the weights' type in the products
  // the n-th of NRF fragments of sub-step s into buffer b: x's, then the weights'
  constexpr int NRF = TM + TN;
  auto read_frag = [&](int slot, int s, int b, int n) {
    const char *st = ring + slot * T::STAGE;
    if (n >= TM) {
      const int j = n - TM;
      if constexpr (T::PACKED) wf[b][j] = *reinterpret_cast<const u32x4_t *>(st + wat[s & 1] + wtile(j) * 64);
      else wf[b][j] = mx_values8<WT>(wraw[j][s], wsc[0][j]);
      return;
    }
#pragma unroll
    for (int e = 0; e < XP; ++e)
      xf[b][n].v[e] = *reinterpret_cast<const u32x4_t *>(st + xat[(XP * s + e) % XPC] + n * 32 * T::XROW);
  };
  f32x16_t acc[TN][TM];
  // The products of sub-step s, from buffer b, in a fixed order, other(n) behind the n-th: LDS reads and direct loads go
  // between them, so that neither the LDS nor the matrix core waits for a burst of the other. Each accumulator passes an
  // empty statement that the compiler may not move: it would else sink a sub-step's products below the barrier, past the
  // reads.
  constexpr int NP = TM * TN;
  auto products = [&](auto sub, int b, auto other) {
    constexpr int S = decltype(sub)::value;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      u32x4_t x[3];
      if constexpr (T::XF32) {
        const u32x4_t a = xf[b][i].v[0], c = xf[b][i].v[XP - 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Split3 q = e < 2 ? split3_bf16(__uint_as_float(a[2 * e]), __uint_as_float(a[2 * e + 1]))
                                 : split3_bf16(__uint_as_float(c[2 * e - 4]), __uint_as_float(c[2 * e - 3]));
          x[0][e] = q.t1;
          x[1][e] = q.t2;
          x[2][e] = q.t3;
        }
      } else {
        x[0] = xf[b][i].v[0];
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const u32x4_t w = wf[b][j];
        if constexpr (T::PACKED) {
          const i32x8_t av = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
          const i32x8_t bv = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], 0, 0, 0, 0};
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc[j][i], 4, 4, S, (int)wsc[0][j], S, (int)xsc[0][i]);
        } else if constexpr (std::is_same_v<X, F16>) {
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, w), __builtin_bit_cast(f16x8_t, x[0]),
                                                             acc[j][i], 0, 0, 0);
        } else {
#pragma unroll
          for (int e = T::XF32 ? 2 : 0; e >= 0; --e)  // smallest terms first
            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, w), __builtin_bit_cast(bf16x8_t, x[e]),
                                                                acc[j][i], 0, 0, 0);
        }
        asm volatile("" : "+v"(acc[j][i]));
        other(i * TN + j);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // the share of `count` operations that goes behind the n-th of `products`, two at a time at least
  auto share = [&](int n, int products, int count, auto &&op) {
    const int each = (count + products - 1) / products > 2 ? (count + products - 1) / products : 2;
#pragma unroll
    for (int o = 0; o < each; ++o)
      if (n * each + o < count) op(n * each + o);
  };
  constexpr auto c_0 = std::integral_constant<int, 0>{};
  constexpr auto c_1 = std::integral_constant<int, 1>{};
  constexpr auto c_2 = std::integral_constant<int, 2>{};

  int slot = 0, tile = 0;  // slot of the stage in use; tiles done
  for (int i = t; i < (PERSIST ? 2 : 1) * T::BN; i += 64 * T::NW) reinterpret_cast<float *>(ring + T::BIAS)[i] = 0.f;
  lds_barrier();
  load_tile();
#pragma unroll
  for (int st = 0; st < NS - 1; ++st) {
#pragma unroll
    for (int n = 0; n < T::OPS; ++n) issue(n, st);
    advance();
  }
  __builtin_amdgcn_s_waitcnt(waitcnt_vm(PERSIST ? 0 : (NS - 2) * T::OPS));  // stage 0 landed (PERSIST: all)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  if (tail && nk == 1) zero_tail(0);
#pragma unroll
  for (int n = 0; n < NRS; ++n) read_stage(0, kg, n, 0);
#pragma unroll
  for (int n = 0; n < NRF; ++n) read_frag(0, 0, 0, n);

  // Stage kt of the tile, in slot SL: a constant, so that LDS addresses are a lane's base and an immediate. (With the slot
  // in a register a stage took 60 instructions more, which bound the small tiles.)
  auto stage = [&](int kt, auto sl) {
    constexpr int SL = decltype(sl)::value, NX = (SL + 1) % NS, TO_SLOT = (SL + NS - 1) % NS;
    const int next = kt + 1 < nk ? kt + 1 : 0;  // PERSIST: the next tile's first
    // the slot refilled here was last read a stage ago, before that stage's barrier
    products(c_0, 0, [&](int n) {
      share(n, NP, NRF + T::OPS, [&](int o) {
        if (o < NRF) read_frag(SL, 1, 1, o);
        else issue(o - NRF, TO_SLOT);
      });
    });
    advance();
    if constexpr (T::SUB == 4) {
      products(c_1, 1, [&](int n) { share(n, NP, NRF, [&](int o) { read_frag(SL, 2, 0, o); }); });
      products(c_2, 0, [&](int n) { share(n, NP, NRF, [&](int o) { read_frag(SL, 3, 1, o); }); });
    }
    // The next stage landed (only those issued after it may be in flight), this wavefront's reads of this one are done;
    // then every one's. PERSIST, first stage of a tile: what is older than its stores was waited for before them.
    if (PERSIST && kt == 0) __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(63));
    else __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((NS - 2) * T::OPS));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (tail && next + 1 == nk) zero_tail(NX);
    // the scales of the stage in use stay until its last products
    products(std::integral_constant<int, T::SUB - 1>{}, 1, [&](int n) {
      share(n, NP, NRS + NRF, [&](int o) {
        if (o < NRS) read_stage(NX, next * KG + kg, o, T::PACKED ? 1 : 0);
        else read_frag(NX, 0, 0, o - NRS);
      });
    });
    if constexpr (T::PACKED) {
#pragma unroll
      for (int j = 0; j < TN; ++j) wsc[0][j] = wsc[1][j];
#pragma unroll
      for (int i = 0; i < TM; ++i) xsc[0][i] = xsc[1][i];
    }
  };

  do {
    place(lid, m0, c0);
    // the sums start as the biases (zeros where there are none, and in the groups of wavefronts that add theirs to group 0's)
    const float *const bias = reinterpret_cast<const float *>(ring + T::BIAS + (PERSIST ? (tile & 1) * T::BN * 4 : 0)) + wn * T::TO * 32 + 4 * h;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 b = *reinterpret_cast<const float4 *>(bias + wtile(j) + 8 * q);
          acc[j][i][4 * q] = b.x;
          acc[j][i][4 * q + 1] = b.y;
          acc[j][i][4 * q + 2] = b.z;
          acc[j][i][4 * q + 3] = b.w;
        }

    // the stages in turn; a tile may end, and the next begin, at any slot
    int kt = 0;
    auto turn = [&](auto sl) {
      constexpr int SL = decltype(sl)::value;
      if (kt < nk && slot == SL) {
        stage(kt, sl);
        ++kt;
        slot = (SL + 1) % NS;
      }
    };
    while (kt < nk) for_each_slot(turn, std::make_integer_sequence<int, NS>{});

    // Epilogue. Lane holds outputs 8 q + 4 h .. + 3 of weight tile j for row l32 of x tile i: activation and product in f32,
    // one rounding, 32 rows x 128 bytes of the wavefront's outputs at a time through LDS (rows padded by 16 bytes), 16-byte
    // pieces out, 8 lanes a row's line. y is written once: not kept in the caches (16392 x 2048 -> 8192: 220 -> 197 us).
    if constexpr (!PERSIST) {
      __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));  // the trailing reloads and reads
      __builtin_amdgcn_s_barrier();                     // every wavefront is done with the ring
    }
    if constexpr (KG > 1) {
      // the groups' sums in group order, through their rings
      float *const part = reinterpret_cast<float *>(ring) + wave * (T::PART / 4);
      if (kg > 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) part[((j * TM + i) * 16 + e) * 64 + lane] = acc[j][i][e];
      }
      lds_barrier();
      if (kg > 0) return;
#pragma unroll
      for (int g = 1; g < KG; ++g)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] += part[g * (T::RING / 4) + ((j * TM + i) * 16 + e) * 64 + lane];
    }
    char *const reg = ring + T::OUT_AT + wave * 32 * T::OROW;
    auto write = [&](auto bytes, auto erf) {
      constexpr bool ERF = decltype(erf)::value;
      constexpr int B = decltype(bytes)::value, JP = 4 / B, EPC = 16 / B;  // output tiles a pass; values of a piece
      constexpr int WIDTH = T::TO < JP ? T::TO * 32 : JP * 32;            // outputs of a pass
      const bool whole = (uintptr_t)p.y % 16 == 0 && p.ldy * B % 16 == 0;
      const bool inside = whole && m0 + T::BM <= p.M && c0 + T::BNO <= p.N;  // uniform: every piece is stored
      char *const ytile = reinterpret_cast<char *>(p.y) + (m0 * p.ldy + c0) * B;
      const uint32_t row8 = (uint32_t)(8 * p.ldy * B);                    // 8 rows of y; a tile spans less than 2^31 bytes
      const uint32_t yoff = (uint32_t)(((wm * TM * 32 + (lane >> 3)) * p.ldy + wn * T::WC + (lane & 7) * EPC) * B);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j0 = 0; j0 < T::TO; j0 += JP) {
#pragma unroll
          for (int jj = 0; jj < JP; ++jj) {
            const int j = j0 + jj;
            if (j >= T::TO) break;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[e] = acc[j][i][4 * q + e];
                if constexpr (ERF) v[e] *= mx_gelu_erf(acc[j + T::TO][i][4 * q + e]);
                else if constexpr (GATED) v[e] *= mx_activate(act, acc[j + T::TO][i][4 * q + e]);
              }
              char *to = reg + l32 * T::OROW + (jj * 32 + 8 * q + 4 * h) * B;
              if constexpr (B == 4) *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
              else if (p.y_dt == LUX3D_BF16) *reinterpret_cast<uint2 *>(to) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
              else *reinterpret_cast<uint2 *>(to) = make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
            }
          }
          // the wavefront's own memory: its LDS operations keep their order, only the compiler has to know
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          // the next tile's stages on their way, before the first store
          if (PERSIST && i == 0 && j0 == 0) __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
          const bool mine = WIDTH * B == 128 || (lane & 7) * 16 < WIDTH * B;
          if (inside) {
#pragma unroll
            for (int it = 0; it < 4; ++it)
              if (mine) st16(ytile + (i * 4 + it) * (uint64_t)row8 + j0 * 32 * B + yoff,
                             *reinterpret_cast<const uint4 *>(reg + (it * 8 + (lane >> 3)) * T::OROW + (lane & 7) * 16));
          } else if (whole) {
#pragma unroll
            for (int it = 0; it < 4; ++it) {
              const int64_t row = m0 + (wm * TM + i) * 32 + it * 8 + (lane >> 3), col = c0 + wn * T::WC + j0 * 32 + (lane & 7) * EPC;
              if (row >= p.M || col >= p.N || !mine) continue;
              const uint4 v = *reinterpret_cast<const uint4 *>(reg + (it * 8 + (lane >> 3)) * T::OROW + (lane & 7) * 16);
              char *dst = ytile + (i * 4 + it) * (uint64_t)row8 + j0 * 32 * B + yoff;
              if (col + EPC <= p.N) {
                st16(dst, v);
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
          } else {
            // rows of y that are not 16-byte aligned: an element a lane, neighbouring lanes in a row
            constexpr int L = WIDTH < 64 ? WIDTH : 64;
            for (int r = lane / L; r < 32; r += 64 / L) {
              const int64_t row = m0 + (wm * TM + i) * 32 + r, col = c0 + wn * T::WC + j0 * 32 + lane % L;
              if (row >= p.M || col >= p.N) continue;
              const char *from = reg + r * T::OROW + (lane % L) * B;
              if constexpr (B == 4) reinterpret_cast<uint32_t *>(p.y)[row * p.ldy + col] = *reinterpret_cast<const uint32_t *>(from);
              else reinterpret_cast<uint16_t *>(p.y)[row * p.ldy + col] = *reinterpret_cast<const uint16_t *>(from);
            }
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
    };
    // f32 erf GELU's form costs 1 to 3% of a call (1029 x 1024 -> 4096 f32 51.1 -> 52.4 us, 4098 x 2048 -> 8192 in 4 bits 107.1 ->
    // 110.5); chosen here, not in the loop (100 x 1024 -> 4096 17.2 us against 18.2).
    if (p.y_dt != LUX3D_F32) write(std::integral_constant<int, 2>{}, std::false_type{});
    else if (GATED && p.act == ACT_GELU_ERF) write(std::integral_constant<int, 4>{}, std::bool_constant<GATED>{});
    else write(std::integral_constant<int, 4>{}, std::false_type{});
    ++tile;
    lid += step;
  } while (PERSIST && lid < end);
  if constexpr (PERSIST) {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));  // the trailing reloads
    if (p.rest > 0)
      for (int64_t share = blockIdx.x; share * 32 < p.N; share += gridDim.x) {
        __syncthreads();
        few_rows((int)share);
      }
  }
}

template <typename X, int WM, int WN, int TM, int TN, int NS, int KG, bool PERSIST, bool GATED>
hipError_t launch_tile(const MxLinearParams &p, hipStream_t s) {
  using T = MxTile<X, WM, WN, TM, TN, NS, KG, PERSIST, GATED>;
  const int64_t tiles_m = (p.M + T::BM - 1) / T::BM, tiles_n = (p.N + T::BNO - 1) / T::BNO;
  const int64_t tiles = tiles_m * tiles_n, cus = PERSIST ? cu_count(s) : tiles;
  const int64_t grid = PERSIST ? (tiles < cus ? tiles : cus) : tiles + (p.rest > 0 ? (p.N + 31) / 32 : 0);
  if (tiles > INT32_MAX || grid * 64 * T::NW * KG > UINT32_MAX) return hipErrorInvalidValue;  // a launch's work-items
  hipLaunchKernelGGL((mx_gemm_kernel<X, WM, WN, TM, TN, NS, KG, PERSIST, GATED>), dim3((unsigned)grid), dim3(64 * T::NW * KG), 0, s, p,
                     mx_act(p.act), (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <typename X, bool GATED>
hipError_t launch_gemm(const MxLinearParams &p, const MxTileId &t, hipStream_t s) {
  const auto is = [&](int rows, int cols, int groups) { return t.rows == rows && t.cols == cols && t.groups == groups; };
  if constexpr (std::is_void_v<X>) {
    if constexpr (!GATED) {
      if (is(64, 64, 1)) return launch_tile<X, 2, 2, 1, 1, 4, 1, false, GATED>(p, s);
      if (is(64, 64, 2)) return launch_tile<X, 2, 2, 1, 1, 4, 2, false, GATED>(p, s);
    }
    if (is(64, 128, 1)) return launch_tile<X, 2, 2, 1, 2, 4, 1, false, GATED>(p, s);
    if (is(128, 128, 1)) return launch_tile<X, 2, 2, 2, 2, 4, 1, false, GATED>(p, s);
    // its bias buffers and waits need four stages a tile
    if (is(256, 256, 1) && p.K > 384) return launch_tile<X, 4, 2, 2, 4, 3, 1, true, GATED>(p, s);
  } else if constexpr (!std::is_same_v<X, F32>) {
    if constexpr (!GATED) {
      if (is(64, 64, 1)) return launch_tile<X, 2, 2, 1, 1, 4, 1, false, GATED>(p, s);
      if (is(64, 64, 2)) return launch_tile<X, 2, 2, 1, 1, 4, 2, false, GATED>(p, s);
      if (is(64, 64, 4)) return launch_tile<X, 2, 2, 1, 1, 3, 4, false, GATED>(p, s);
    }
    if (is(64, 128, 1)) return launch_tile<X, 2, 2, 1, 2, 4, 1, false, GATED>(p, s);
    if (is(64, 128, 2)) return launch_tile<X, 2, 2, 1, 2, 4, 2, false, GATED>(p, s);
    if (is(64, 128, 4)) return launch_tile<X, 2, 2, 1, 2, 3, 4, false, GATED>(p, s);
    if (is(128, 128, 1)) return launch_tile<X, 2, 2, 2, 2, 3, 1, false, GATED>(p, s);
    // two wavefronts a SIMD (four of 64 x 128 in all: 4096 rows of 8192 -> 2048 122 us against 118)
    if (is(128, 256, 1)) return launch_tile<X, 2, 4, 2, 2, 3, 1, false, GATED>(p, s);
    if (is(256, 256, 1)) return launch_tile<X, 2, 4, 4, 2, 3, 1, false, GATED>(p, s);
  } else {
    // a wavefront's 32 rows of x meet 128 weight rows, so that each value is split into its three terms once a workgroup
    // (64 x 64 a wavefront, 4100 rows of 8192 -> 2048: 472 us against 397)
    if constexpr (!GATED)
      if (is(64, 64, 4)) return launch_tile<X, 2, 2, 1, 1, 4, 4, false, GATED>(p, s);
    if (is(64, 128, 2)) return launch_tile<X, 2, 1, 1, 4, 3, 2, false, GATED>(p, s);
    if (is(64, 128, 4)) return launch_tile<X, 2, 1, 1, 4, 3, 4, false, GATED>(p, s);
  }
  return hipErrorInvalidValue;
}

template <typename X>
hipError_t launch_gemm(const MxLinearParams &p, const MxTileId &t, hipStream_t s) {
  return p.act >= 0 ? launch_gemm<X, true>(p, t, s) : launch_gemm<X, false>(p, t, s);
}

}  // namespace

hipError_t launch_mx_gemm(const MxLinearParams &p, const MxTileId &t, hipStream_t s) {
  if (!p.x) return launch_gemm<void>(p, t, s);
  switch (p.x_dt) {
    case LUX3D_F32: return launch_gemm<F32>(p, t, s);
    case LUX3D_BF16: return launch_gemm<BF16>(p, t, s);
    case LUX3D_F16: return launch_gemm<F16>(p, t, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lux3d
