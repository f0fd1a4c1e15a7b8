// prefix_attention.hip -- attention of a batch whose sequences share one long prefix of keys:
//   out[b, h, i] = softmax over the P prefix keys and the own keys j that query i sees of (q . k * scale), times v
// An own key j is seen when j < len_b and, with causality, j <= len_b - Lq + i. The prefix's K and V exist once, for all
// sequences; a head group of H / Hkv query heads shares a key head.
//
// What bounds it. Long queries: the matrix cores, 4 D operations a visible (query, key) pair. Decoding: the bytes of K
// and V. The rows that share a key head's prefix, of all sequences and of the group's heads, are therefore taken
// together, 128 rows a tile: the prefix is read once for up to 128 of them instead of once a row. Own keys are read by
// workgroups of their own. Every workgroup takes a run of key blocks, so that few rows still fill the chip, and leaves
// an unnormalised partial result (maximum, sum, O); a second kernel merges a row's partials in their order.
//
// Numerics: f32 scores, softmax with a running maximum and sums in f32. The 2-byte types' probabilities are rounded to
// the type for P v (the row sum adds the rounded ones), as lux3d_sdpa does: the matrix instructions take 2-byte operands,
// and two terms a probability would double the product. Error against 64 bits, with / without that rounding: 0.0023 /
// 0.0017 of the output's norm in bf16, 0.00029 / 0.00021 in f16. out is rounded once. A row that sees no key is zero.
//
// Masks. Keys past a sequence's length are never read: the buffer loads end at the last visible key and return zeros, so
// that a probability of zero meets a finite value. Inside a tile, keys that causality hides from some of its rows are
// read for the others: their scores become -inf whatever K holds, and their V, times a probability of zero, has to be
// finite.
#include <type_traits>

#include "attn_tiles.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace lux3d {

namespace {

__device__ __forceinline__ int64_t own_len(const PrefixParams &p, int64_t b) {
  int64_t n = p.lens ? p.lens[b] : p.Ls;
  n = n < 0 ? 0 : n;
  return n < p.Ls ? n : p.Ls;
}
// own keys that query i of a sequence of `len` sees
__device__ __forceinline__ int64_t own_seen(const PrefixParams &p, int64_t len, int64_t i) {
  if (!p.causal) return len;
  const int64_t n = len - p.Lq + i + 1;
  return n < 0 ? 0 : n;
}

// The rows and keys of a workgroup. Rows r0 .. rlim - 1 of key head kv (b * R + i * group + head in the group); keys
// p0 .. p1 of the prefix and o0 .. o1 of sequence b.
struct PrefixItem {
  int64_t kv, r0, rlim, b;
  int64_t p0, p1, o0, o1;
  int64_t part;
};

// `first`: joint items and prefix items, else own items (lid counts each kind from 0)
__device__ __forceinline__ PrefixItem prefix_item(const PrefixParams &p, int64_t lid, bool first) {
  const PrefixPlan &s = p.plan;
  const int64_t R = p.Lq * p.G;
  uint32_t x = (uint32_t)lid;
  PrefixItem w;
  w.p0 = w.p1 = w.o0 = w.o1 = w.b = 0;
  int tile = s.tile;
  if (first && !s.joint) {
    // tiles innermost: those that share keys run side by side
    const uint32_t tiles = (uint32_t)s.prefix_tiles, runs = (uint32_t)s.prefix_runs;
    const uint32_t t = x % tiles;
    x /= tiles;
    w.part = x % runs;
    w.kv = x / runs;
    w.r0 = (int64_t)t * tile;
    w.rlim = p.B * R;
    const int64_t run = s.prefix_run * kPrefixKeys;
    w.p0 = w.part * run;
    w.p1 = w.p0 + run < p.P ? w.p0 + run : p.P;
    return w;
  }
  if (s.joint) {
    // key heads outermost: the tiles of one XCD share a key head's prefix in its L2
    const uint32_t tiles = (uint32_t)s.own_tiles, B = (uint32_t)p.B, runs = (uint32_t)s.own_runs;
    const uint32_t t = x % tiles;
    x /= tiles;
    w.b = x % B;
    x /= B;
    w.part = x % runs;
    w.kv = x / runs;
    w.r0 = w.b * R + (int64_t)t * tile;
    // blocks of the prefix, then of the own keys, in runs
    const int64_t pb = (p.P + kPrefixKeys - 1) / kPrefixKeys;
    const int64_t j0 = w.part * s.own_run, j1 = j0 + s.own_run;
    w.p0 = j0 * kPrefixKeys;
    w.p1 = j1 * kPrefixKeys < p.P ? j1 * kPrefixKeys : p.P;
    w.o0 = j0 > pb ? (j0 - pb) * kPrefixKeys : 0;
    w.o1 = j1 > pb ? (j1 - pb) * kPrefixKeys : 0;
  } else {
    tile = s.own_tile;
    const uint32_t tiles = (uint32_t)s.own_tiles, runs = (uint32_t)s.own_runs, hkv = (uint32_t)p.Hkv;
    const uint32_t t = x % tiles;
    x /= tiles;
    const uint32_t pr = x % runs;
    x /= runs;
    w.kv = x % hkv;
    w.b = x / hkv;
    w.part = s.prefix_runs + pr;
    w.r0 = w.b * R + (int64_t)t * tile;
    w.o0 = pr * s.own_run * kPrefixKeys;
    w.o1 = w.o0 + s.own_run * kPrefixKeys;
  }
  w.rlim = (w.b + 1) * R;
  if (w.o1 > w.o0) {  // up to what the tile's last query sees
    const int64_t last = (w.r0 + tile < w.rlim ? w.r0 + tile : w.rlim) - 1;
    const int64_t seen = own_seen(p, own_len(p, w.b), (last - w.b * R) / p.G);
    w.o1 = w.o1 < seen ? w.o1 : seen;
  }
  if (w.p1 < w.p0) w.p1 = w.p0;
  if (w.o1 < w.o0) w.o1 = w.o0;
  w.o1 = uniform(w.o1);
  return w;
}

// Row g of key head kv as (sequence, position, query head).
struct PrefixRow {
  int64_t b, i, h;
};
__device__ __forceinline__ PrefixRow prefix_row(const PrefixParams &p, int64_t kv, int64_t g) {
  const uint32_t R = (uint32_t)(p.Lq * p.G), G = (uint32_t)p.G, x = (uint32_t)g;
  const uint32_t b = x / R, r = x - b * R, i = r / G;
  return {(int64_t)b, (int64_t)i, kv * p.G + (int64_t)(r - i * G)};
}

// Few rows in the 2-byte types. Four wavefronts: two row groups of 32 rows, the KS = 2 wavefronts of a group taking 32 of
// every block's 64 keys each. S^T = K Q^T, O^T += V^T P^T as attn_mfma_kernel does it: each lane holds one row's
// scores of 16 keys, K and V blocks come by direct global -> LDS loads, two blocks deep.
template <int D> struct PrefixLds {
  // the ring of two K and two V blocks; at the end the key groups' partial results
  static constexpr int PW = (D / 32 * 16 + 2) * 64;  // floats of a wavefront
  static constexpr int bytes = 4 * kPrefixKeys * D * 2 > 4 * PW * 4 ? 4 * kPrefixKeys * D * 2 : 4 * PW * 4;
};
template <typename T, int D>
__device__ __forceinline__ void prefix_attend(const PrefixParams &p, const PrefixItem &w, uint16_t *smem) {
  using M = Mma<T>;
  using op_t = typename M::op_t;
  constexpr int KS = 2, BKV = kPrefixKeys, NDT = D / 32;
  constexpr int KCH = BKV * D / 8 / 256;   // 16-byte chunks of K (and V) per thread and block
  constexpr int BUF = BKV * D;             // 2-byte elements of a block
  constexpr bool VEARLY = D == 128;        // V's fragments before the softmax
  constexpr int PW = PrefixLds<D>::PW;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int qg = wave / KS, kg = wave % KS;  // kg: the block's 32 keys, too

  const int64_t g = w.r0 + qg * 32 + l32;          // this lane's row
  const bool live = g < w.rlim;
  const bool rows = w.r0 + qg * 32 < w.rlim;       // this wavefront's row group has rows (uniform)
  const int np = (int)((w.p1 - w.p0 + BKV - 1) / BKV), no = (int)((w.o1 - w.o0 + BKV - 1) / BKV), nblk = np + no;

  op_t qf[D / 16];
  int seen;  // own keys that this lane's row sees; all_seen: that every row of the tile sees (blocks below need no mask)
  int all_seen;
  {
    const PrefixRow row = prefix_row(p, w.kv, live ? g : w.rlim - 1);
    const int64_t len = own_len(p, w.b);
    seen = (int)own_seen(p, len, row.i);
    all_seen = __builtin_amdgcn_readfirstlane((int)own_seen(p, len, (w.r0 - w.b * p.Lq * p.G) / p.G));
    const char *q = reinterpret_cast<const char *>(p.q) + (row.b * p.q_sb + row.h * p.q_sh + row.i * p.q_st) * 2;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const op_t *>(q + (c * 16 + 8 * hh) * 2);
  }

  // direct loads: load i of a wavefront fills 1 KB of a block in lane order; a lane's slot holds the row's chunk that the
  // swizzle puts there. Descriptors start at the block's first key and end at the range's last: beyond it zeros.
  const char *pk = reinterpret_cast<const char *>(p.pk) + w.kv * p.pk_sh * 2;
  const char *pv = reinterpret_cast<const char *>(p.pv) + w.kv * p.pv_sh * 2;
  const char *ok = reinterpret_cast<const char *>(p.k) + (w.b * p.k_sb + w.kv * p.k_sh) * 2;
  const char *ov = reinterpret_cast<const char *>(p.v) + (w.b * p.v_sb + w.kv * p.v_sh) * 2;
  const uint32_t lds_k = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t *)smem;
  const uint32_t lds_v = lds_k + 2 * BUF * 2;
  // row and slot of the lane's first load; load i's row is RS i further on, its row bits disjoint from r0's in the swizzle
  constexpr int RS = 512 / D;
  const int r0 = wave * KCH * RS + lane / (D / 8);
  uint32_t row0 = (uint32_t)r0, kch = (uint32_t)(((lane % (D / 8)) ^ k_swz<D>(r0)) * 16);
  const uint32_t vch = (uint32_t)(((lane % (D / 8)) ^ v_swz<D>(r0)) * 16);
  auto issue = [&](int j, int buf) {
    const bool pre = j < np;
    const int64_t key0 = pre ? w.p0 + (int64_t)j * BKV : w.o0 + (int64_t)(j - np) * BKV;
    const int64_t rest = (pre ? w.p1 : w.o1) - key0;
    const int left = rest < BKV ? (int)rest : BKV;    // keys of this block, >= 1
    const int64_t kst = pre ? p.pk_st : p.k_st, vst = pre ? p.pv_st : p.v_st;
    const i32x4_t krs = buffer_rsrc((pre ? pk : ok) + key0 * kst * 2, ((left - 1) * kst + D) * 2);
    const i32x4_t vrs = buffer_rsrc((pre ? pv : ov) + key0 * vst * 2, ((left - 1) * vst + D) * 2);
    const uint32_t ks2 = (uint32_t)kst * 2, vs2 = (uint32_t)vst * 2;
    asm volatile("" : "+v"(row0), "+v"(kch));  // formed here, not kept across the loop
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const uint32_t off = (uint32_t)((wave * KCH + i) * 1024 + buf * BUF * 2);
      lds_load16(krs, row0 * ks2 + i * RS * ks2 + (kch ^ (k_swz<D>(i * RS) * 16)), 0,
                 __builtin_amdgcn_readfirstlane(lds_k + off));
      lds_load16(vrs, row0 * vs2 + i * RS * vs2 + vch, 0, __builtin_amdgcn_readfirstlane(lds_v + off));
    }
  };

  f32x16_t o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16_t{};
  float m = -INFINITY, l = 0.f;
  const float c2 = p.scale * kLog2e;

  auto step = [&](int j, auto mask_c) {
    constexpr bool MASK = decltype(mask_c)::value;
    const int buf = j & 1;
    if (j + 1 < nblk) issue(j + 1, buf ^ 1);
    if (!rows) {  // a row group past the tile's last row only loads
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      lds_barrier();
      return;
    }
    const uint16_t *Ks = smem + buf * BUF, *Vs = smem + 2 * BUF + buf * BUF;
    f32x16_t s = f32x16_t{};
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const int krow = kg * 32 + l32;
      const op_t a = *reinterpret_cast<const op_t *>(Ks + krow * D + ((2 * c + hh) ^ k_swz<D>(krow)) * 8);
      s = M::run(a, qf[c], s);
    }
    // this lane's row sees keys below lim of the block; lane holds keys 8 (i / 4) + 4 hh + i % 4 of its 32
    int lim = BKV;
    if constexpr (MASK) {
      lim = j < np ? (int)(w.p1 - w.p0) - j * BKV : seen - (int)w.o0 - (j - np) * BKV;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kg * 32 + 8 * (i >> 2) + (i & 3) >= lim - 4 * hh) s[i] = -INFINITY;
    }
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
    // V^T fragment of dim tile dt, keys 16 jj ..: see attn_mfma_kernel
    auto vfrag = [&](int dt, int jj) {
      const int g16 = lane & 15;
      const int vrow = kg * 32 + 16 * jj + 4 * hh + (g16 >> 2);
      const int vcol = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (g16 & 3);
      const uint16_t *vr = Vs + vrow * D + ((vcol >> 3) ^ v_swz<D>(vrow)) * 8 + (vcol & 7);
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vr));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vr + 8 * D));
      return __builtin_bit_cast(op_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // V's fragments are read before the softmax, which hides their latency
    op_t vf[VEARLY ? NDT * 2 : 1];
    if constexpr (VEARLY) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) vf[dt * 2 + jj] = vfrag(dt, jj);
      __builtin_amdgcn_sched_barrier(0);
    }

    // running maximum: it moves when a block's exceeds it by 2^8, so that most blocks need no rescale
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
    const float cand = half_swap_max(mx) * c2;
    const float mn = cand > m + 8.f ? cand : m;
    const float mb = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every probability is exp2(-inf)
    const float alpha = __builtin_amdgcn_exp2f(m - mb);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
    }
    m = mn;
    op_t pf[2];
    float ls = 0.f;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      u32x4_t pk4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * jj + 2 * e], c2, -mb));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * jj + 2 * e + 1], c2, -mb));
        pk4[e] = M::pack(p0, p1);
        ls = M::sum2(pk4[e], ls);
      }
      pf[jj] = __builtin_bit_cast(op_t, pk4);
    }
    l = l * alpha + ls;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) o[dt] = M::run(VEARLY ? vf[dt * 2 + jj] : vfrag(dt, jj), pf[jj], o[dt]);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // this wavefront's part of block j + 1 landed
    lds_barrier();
  };

  if (nblk > 0) {
    issue(0, 0);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
    for (int j = 0; j < nblk; ++j) {
      const bool whole = j < np ? w.p0 + (int64_t)(j + 1) * BKV <= w.p1 : w.o0 + (int64_t)(j - np + 1) * BKV <= all_seen;
      if (whole) step(j, std::false_type{});
      else step(j, std::true_type{});
    }
  }

  // a row group's KS partial results, through LDS in key-group order; wavefront kg keeps the dim tiles dt % KS == kg
  float *part = reinterpret_cast<float *>(smem), *mine = part + wave * PW;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) mine[(dt * 16 + i) * 64 + lane] = o[dt][i];
  mine[NDT * 16 * 64 + lane] = m;
  mine[(NDT * 16 + 1) * 64 + lane] = l;
  lds_barrier();
  const float *grp = part + qg * KS * PW;
  float a[KS], mm = -INFINITY;
#pragma unroll
  for (int k2 = 0; k2 < KS; ++k2) mm = fmaxf(mm, grp[k2 * PW + NDT * 16 * 64 + lane]);
  const float mb = mm == -INFINITY ? 0.f : mm;
  l = 0.f;
#pragma unroll
  for (int k2 = 0; k2 < KS; ++k2) {
    a[k2] = __builtin_amdgcn_exp2f(grp[k2 * PW + NDT * 16 * 64 + lane] - mb);
    l += grp[k2 * PW + (NDT * 16 + 1) * 64 + lane] * a[k2];
  }
  m = mm;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    if (dt % KS != kg) continue;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = 0.f;
#pragma unroll
      for (int k2 = 0; k2 < KS; ++k2) acc += grp[k2 * PW + (dt * 16 + i) * 64 + lane] * a[k2];
      o[dt][i] = acc;
    }
  }

  const float total = half_swap_sum(l);
  if (!live) return;
  // lane holds dims dt * 32 + 8 g4 + 4 hh + {0..3}, g4 = 0..3
  if (p.plan.parts > 1) {
    const int64_t rows = p.B * p.Lq * p.G * p.Hkv, r = (w.part * p.Hkv + w.kv) * (p.B * p.Lq * p.G) + g;
    float *po = p.ws + r * D;
    if (kg == 0 && hh == 0) *reinterpret_cast<float2 *>(p.ws + p.plan.parts * rows * D + r * 2) = make_float2(m, total);
    if (m == -INFINITY) return;  // no key seen: the merge does not take this part's O
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      if (dt % KS != kg) continue;
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<float4 *>(po + dt * 32 + 8 * g4 + 4 * hh) =
            make_float4(o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]);
    }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const PrefixRow row = prefix_row(p, w.kv, g);
  char *orow = reinterpret_cast<char *>(p.o) + (row.b * p.o_sb + row.h * p.o_sh + row.i * p.o_st) * 2;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) {
    if (dt % KS != kg) continue;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<uint2 *>(orow + (dt * 32 + 8 * g4 + 4 * hh) * 2) =
          make_uint2(M::pack(o[dt][4 * g4] * inv, o[dt][4 * g4 + 1] * inv),
                     M::pack(o[dt][4 * g4 + 2] * inv, o[dt][4 * g4 + 3] * inv));
  }
}

// ---- pipelined form: 128 rows a workgroup ----------------------------------------
//
// attn_pipe_kernel's pipeline over the blocks of two key ranges: keys go by 32, two steps to a pair, and step j is one
// straight line of MFMAs (scores of block j + 2, O += P V of block j) with the exponentials, the maximum and the LDS reads
// in the gaps between them. Each of the 4 wavefronts keeps 32 rows. A block lies in one range: the prefix's
// last one ends where the prefix ends, and the next begins the own keys. K and V arrive by direct global -> LDS loads in
// two stages of 64 keys, of which wavefronts 0 and 1 load the first block and 2 and 3 the second, so that each builds the
// descriptor of its block's range; what lies past the range reads as zeros.
// The running maximum starts at -3e38 rather than -inf: a row that has seen nothing yet forms exp2(-inf) = 0.
template <typename T, int D>
__device__ __forceinline__ void prefix_attend_pipe(const PrefixParams &p, const PrefixItem &w, char *ring, int *seen_lds) {
  using M = Mma<T>;
  using op_t = typename M::op_t;
  constexpr int BK = 32, NC = D / 16, NDT = D / 32;
  constexpr int KB = BK * D * 2, STAGE = 4 * KB;          // bytes of a block; a stage: V, V, K, K
  constexpr int SEGW = 2 * KB / 1024 / 4;                 // direct loads per wavefront for two blocks
  constexpr int RS = 512 / D;                             // rows of a load
  static_assert(SEGW * RS == 16, "two wavefronts load a block");
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  int *const seen = seen_lds + wave * 32 + l32;  // own keys from o0 on that the lane's row sees: read for a mask only
  const int np = (int)((w.p1 - w.p0 + BK - 1) / BK), no = (int)((w.o1 - w.o0 + BK - 1) / BK), nkv = np + no;

  op_t qf[NC];
  int all_seen;  // own keys from o0 on that every row of the tile sees
  {
    const int64_t len = own_len(p, w.b);
    all_seen = __builtin_amdgcn_readfirstlane((int)(own_seen(p, len, (w.r0 - w.b * p.Lq * p.G) / p.G) - w.o0));
    const int64_t g = w.r0 + wave * 32 + l32;
    const PrefixRow row = prefix_row(p, w.kv, g < w.rlim ? g : w.rlim - 1);
    *seen = (int)(own_seen(p, len, row.i) - w.o0);
    const char *q = reinterpret_cast<const char *>(p.q) + (row.b * p.q_sb + row.h * p.q_sh + row.i * p.q_st) * 2;
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = *reinterpret_cast<const op_t *>(q + (c * 16 + 8 * hh) * 2);
  }

  // the lane's part of a load: row r0 + RS i of its wavefront's block, the chunk that its slot holds
  uint32_t ln = (uint32_t)lane;  // opaque in each load: its parts are formed again there, not kept
  auto row_of = [&]() { return (uint32_t)(wave & 1) * 16 + ln / (D / 8); };
  const char *ok = reinterpret_cast<const char *>(p.k) + (w.b * p.k_sb + w.kv * p.k_sh + w.o0 * p.k_st) * 2;
  const char *ov = reinterpret_cast<const char *>(p.v) + (w.b * p.v_sb + w.kv * p.v_sh + w.o0 * p.v_st) * 2;
  const int pn = (int)(w.p1 - w.p0), own_end = np * BK + (int)(w.o1 - w.o0);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)ring;
  // The wavefront's blocks of K (of V): the descriptor of block `blk` of the item's, its keys of the range and zeros beyond.
  // A stage's descriptors are formed while the stage before it is worked on, without branches: at the head of a stage, or
  // with a branch for the range, their scalar instructions cost 8 to 15% of the kernel.
  struct Source {
    const char *pre, *own;
    uint32_t pst2, ost2, st2;  // bytes from key to key: of the prefix, of the own keys, of this block
    int blk;
    i32x4_t rs;
  };
  auto describe = [&](Source &s) {
    const bool own = s.blk >= np;
    const int at = s.blk * BK, left = (own ? own_end : pn) - at, rows = left < BK ? left : BK;
    s.st2 = own ? s.ost2 : s.pst2;
    const uint64_t a = (uint64_t)(own ? s.own : s.pre) + (uint64_t)(uint32_t)at * s.st2;
    const int bytes = rows > 0 ? (rows - 1) * (int)s.st2 + 2 * D : 0;
    s.rs = i32x4_t{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)),
                   __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
  };
  auto source = [&](int blk, const void *pre, int64_t sh, int64_t pst, const char *own, int64_t ost) {
    Source s;
    s.pre = reinterpret_cast<const char *>(pre) + (w.kv * sh + w.p0 * pst) * 2;
    s.own = own - (int64_t)(np * BK) * ost * 2;  // as if its blocks had been counted from the item's first
    s.pst2 = (uint32_t)pst * 2;
    s.ost2 = (uint32_t)ost * 2;
    s.blk = blk + (wave >> 1);
    describe(s);
    return s;
  };
  Source sk = source(0, p.pk, p.pk_sh, p.pk_st, ok, p.k_st), sv = source(0, p.pv, p.pv_sh, p.pv_st, ov, p.v_st);
  auto load_k = [&](const Source &s, uint32_t lds) {
    asm volatile("" : "+v"(ln));
    const uint32_t r = row_of(), off = r * s.st2, ch = ((ln % (D / 8)) ^ (uint32_t)k_swz<D>((int)r)) * 16;
#pragma unroll
    for (int i = 0; i < SEGW; ++i)
      lds_load16(s.rs, off + (uint32_t)(i * RS) * s.st2 + (ch ^ (k_swz<D>(i * RS) * 16)), 0,
                 __builtin_amdgcn_readfirstlane(lds + (wave * SEGW + i) * 1024));
  };
  auto load_v = [&](const Source &s, uint32_t lds) {
    asm volatile("" : "+v"(ln));
    const uint32_t r = row_of(), off = r * s.st2 + ((ln % (D / 8)) ^ (uint32_t)v_swz<D>((int)r)) * 16;
#pragma unroll
    for (int i = 0; i < SEGW; ++i)
      lds_load16(s.rs, off + (uint32_t)(i * RS) * s.st2, 0, __builtin_amdgcn_readfirstlane(lds + (wave * SEGW + i) * 1024));
  };
  int slot = 0;  // stage g: V's blocks 2 g, 2 g + 1, K's 2 g + 3, 2 g + 4
  auto load_stage = [&](int to) {
    load_v(sv, lds0 + to * STAGE);
    load_k(sk, lds0 + to * STAGE + 2 * KB);
  };
  int kfo = 2 * KB + l32 * 2 * D + ((hh ^ k_swz<D>(l32)) << 4);
  auto kfrag = [&](int at, int c) { return *reinterpret_cast<const op_t *>(ring + at + (kfo ^ (c << 5))); };
  typedef short s16x4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
  const int vr0 = 4 * hh + ((lane & 15) >> 2), vc0 = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  int vfo = vr0 * 2 * D + (((vc0 >> 3) ^ v_swz<D>(vr0)) << 4) + (vc0 & 7) * 2;
  auto vhalf = [&](int at, int dt, int jj, int h) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4_t *)(ring + at + (vfo ^ (dt << 6)) + (16 * jj + 8 * h) * 2 * D));
  };

  f32x16_t o[NDT], sa, sb;
  float m = -3e38f, l = 0.f, ls = 0.f, alpha, mx;
  op_t kf[NC], pf[2];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16_t{};
  const float c2 = p.scale * kLog2e;

  // block j's keys that a row does not see (past the prefix's end, the sequence's, or by causality) score -inf
  auto mask = [&](int j, f32x16_t &s) {
    const int lim = (j < np ? pn - j * BK : j < nkv ? *seen - (j - np) * BK : 0) - 4 * hh;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (8 * (i >> 2) + (i & 3) >= lim) s[i] = -INFINITY;
  };
  // blocks that need a mask: the prefix's last where it is not whole, and from own_first on
  const int cut = pn % BK ? np - 1 : -1, all = all_seen > 0 ? all_seen / BK : 0, own_first = np + (all < no ? all : no);
  auto partial = [&](int j) { return (j == cut) | (j >= own_first); };
  auto max_step = [&](const f32x16_t &s, int i, bool first) {
    if (first && i == 0) mx = fmaxf(s[0], s[1]);
    else mx = fmaxf(fmaxf(mx, s[2 * i]), s[2 * i + 1]);
  };
  auto max_done = [&]() {
    const float cand = half_swap_max(mx) * c2;
    float mn = m;
    if (cand > mn + 8.f) mn = cand;
    alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
  };
  auto sum_pair = [&]() { l = __builtin_fmaf(l, alpha, ls); };

  if (nkv > 0) {
    // prologue: K's blocks 0, 1 and 2, 3 into the slot of stage 1, stage 0; the scores of the first pair, its maximum
    load_k(sk, lds0 + STAGE + 2 * KB);
    sk.blk += 2;
    describe(sk);
    load_k(sk, lds0 + STAGE);
    sk.blk += 1;
    describe(sk);
    load_stage(0);
    sk.blk += 2;
    sv.blk += 2;
    describe(sk);
    describe(sv);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(2 * SEGW));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    auto scores = [&](f32x16_t &s) {
#pragma unroll
      for (int c = 0; c < NC; ++c) s = M::run(kf[c], qf[c], c == 0 ? f32x16_t{} : s);
    };
#pragma unroll
    for (int c = 0; c < NC; ++c) kf[c] = kfrag(STAGE, c);
    scores(sa);
#pragma unroll
    for (int c = 0; c < NC; ++c) kf[c] = kfrag(STAGE + KB, c);
    scores(sb);
#pragma unroll
    for (int c = 0; c < NC; ++c) kf[c] = kfrag(STAGE - 2 * KB, c);
    mask(0, sa);
    mask(1, sb);
#pragma unroll
    for (int i = 0; i < 8; ++i) max_step(sa, i, true);
#pragma unroll
    for (int i = 0; i < 8; ++i) max_step(sb, i, false);
    max_done();

    // One step on block j, of parity PAR, whose scores are in s. NEXT: there is a next pair, and the scores of block
    // j + 2 replace them. The mask is a branch inside the step: a second form of the step beside it, chosen by the block,
    // spills 157 registers.
    auto step = [&](int j, f32x16_t &s, auto par_c, auto next_c) {
      constexpr int PAR = decltype(par_c)::value;
      constexpr bool NEXT = decltype(next_c)::value;
      // MFMAs: the scores but for their last chunk, one half of P v, the scores' last chunk, the other half
      constexpr int NA = NEXT ? NC - 1 : 0, NL = NEXT ? 1 : 0, NB = 2 * NDT, NM = NA + NB + NL;
      constexpr int LAST = NA + NB / 2;  // the scores' last chunk
      constexpr int at = PAR * KB;
      if constexpr (PAR == 0) {
        // the stage landed, and every wavefront is done with the one before
        __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        load_stage(slot ^ 1);
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
        }
        ls = 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);
      s16x4_t vh[NDT][2][2];
      f32x16_t sn;
      // exponentials, two pairs of scores at a time: 4 FMAs, 4 exponentials, 2 packs, 2 sums
      auto exp_op = [&](int n) {
        const int r = n % 12, e0 = 4 * (n / 12);
        if (r < 4) {
          s[e0 + r] = __builtin_fmaf(s[e0 + r], c2, -m);
        } else if (r < 8) {
          s[e0 + r - 4] = __builtin_amdgcn_exp2f(s[e0 + r - 4]);
        } else {
          const int h = r & 1, pe = e0 / 2 + h;  // packed pair pe of the tile: element pe % 4 of fragment pe / 4
          u32x4_t pk4 = __builtin_bit_cast(u32x4_t, pf[pe / 4]);
          if (r < 10) pk4[pe % 4] = M::pack(s[e0 + 2 * h], s[e0 + 2 * h + 1]);
          else ls = M::sum2(pk4[pe % 4], ls);
          pf[pe / 4] = __builtin_bit_cast(op_t, pk4);
        }
      };
      // VALU items: 4 groups of 12; 8 steps of the maximum and the pair's end
      constexpr int NEXP = 48, NMAX = !NEXT ? 0 : PAR == 1 ? 9 : 8, REST = NB / 2;
      if constexpr (!NEXT) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int jj = 0; jj < 2; ++jj)
#pragma unroll
            for (int h = 0; h < 2; ++h) vh[dt][jj][h] = vhalf(at, dt, jj, h);
#pragma unroll
        for (int n = 0; n < NEXP; ++n) exp_op(n);
      }
#pragma unroll
      for (int u = 0; u < NM; ++u) {
        if (u < NA) {
          sn = M::run(kf[u], qf[u], u == 0 ? f32x16_t{} : sn);
          // V's 4 NDT fragment halves, spread over these MFMAs
#pragma unroll
          for (int x = 0; x < 4 * NDT; ++x)
            if (x >= u * 4 * NDT / (NA ? NA : 1) && x < (u + 1) * 4 * NDT / (NA ? NA : 1))
              vh[x / 4][x / 2 % 2][x % 2] = vhalf(at, x / 4, x / 2 % 2, x % 2);
        } else if (u >= LAST && u < LAST + NL) {
          s = M::run(kf[NC - 1], qf[NC - 1], sn);
          keep(sn);  // the product goes to s's registers, not to sn's and a copy
        } else {
          const int b = u < LAST ? u - NA : u - NA - NL, jj = b / NDT, dt = b % NDT;
          const op_t a = __builtin_bit_cast(op_t, __builtin_shufflevector(vh[dt][jj][0], vh[dt][jj][1], 0, 1, 2, 3, 4, 5, 6, 7));
          o[dt] = M::run(a, pf[jj], o[dt]);
          if (NEXT && b < NC) kf[b] = kfrag(at, b);
        }
        if constexpr (NEXT) {
#pragma unroll
          for (int n = 0; n < NEXP; ++n)
            if (n >= u * NEXP / LAST && n < (u + 1) * NEXP / LAST) exp_op(n);
          if (PAR == 1 && u == LAST - 1) sum_pair();
          if (u == LAST + NL - 1) {
            // formed by here: the compiler would move what is used behind the branch there, away from the MFMAs before it
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) asm volatile("" ::"v"(pf[jj]), "v"(ls), "v"(l));
#pragma unroll
            for (int x = 0; x < 4 * NDT; ++x) asm volatile("" ::"v"(vh[x / 4][x / 2 % 2][x % 2]));
            if (partial(j + 2)) mask(j + 2, s);
          }
          // the next stage's descriptors
          if (PAR == 1 && (u == 1 || u == 3)) {
            Source &src = u == 1 ? sv : sk;
            src.blk += 2;
            describe(src);
          }
          const int r = u - LAST - NL;
#pragma unroll
          for (int n = 0; n < NMAX; ++n)
            if (r >= 0 && n >= r * NMAX / REST && n < (r + 1) * NMAX / REST) {
              if (n < 8) max_step(s, n, PAR == 0);
              else max_done();
            }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (PAR == 1) {
        slot ^= 1;
        kfo ^= STAGE;
        vfo ^= STAGE;
      }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    constexpr std::true_type yes{};
    constexpr std::false_type no_{};
    int j = 0;
    for (; j + 2 < nkv; j += 2) {
      step(j, sa, even, yes);
      step(j + 1, sb, odd, yes);
    }
    step(j, sa, even, no_);
    if (j + 2 == nkv) step(j + 1, sb, odd, no_);
    sum_pair();
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));  // the trailing reloads
  }

  // lane holds dims dt * 32 + 8 g4 + 4 hh + {0..3}, g4 = 0..3
  const int64_t g = w.r0 + wave * 32 + l32;
  const float total = half_swap_sum(l);
  if (g >= w.rlim) return;
  if (p.plan.parts > 1) {
    const int64_t per = p.B * p.Lq * p.G, rows = per * p.Hkv, r = w.part * rows + w.kv * per + g;
    const bool none = total == 0.f;
    if (hh == 0) *reinterpret_cast<float2 *>(p.ws + p.plan.parts * rows * D + r * 2) = make_float2(none ? -INFINITY : m, total);
    if (none) return;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<float4 *>(p.ws + r * D + dt * 32 + 8 * g4 + 4 * hh) =
            make_float4(o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]);
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const PrefixRow row = prefix_row(p, w.kv, g);
  char *orow = reinterpret_cast<char *>(p.o) + (row.b * p.o_sb + row.h * p.o_sh + row.i * p.o_st) * 2;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<uint2 *>(orow + (dt * 32 + 8 * g4 + 4 * hh) * 2) =
          make_uint2(M::pack(o[dt][4 * g4] * inv, o[dt][4 * g4 + 1] * inv),
                     M::pack(o[dt][4 * g4 + 2] * inv, o[dt][4 * g4 + 3] * inv));
}

// JOINT: every workgroup 128 / KS rows (128: pipelined) of one sequence through prefix and own keys. Else pipelined prefix
// items of 128 rows, and own items whose few rows split each block's keys between two wavefronts.
template <typename T, int D, bool JOINT, int KS, int MINW>
__global__ __launch_bounds__(256, MINW) void prefix_attn_kernel(PrefixParams p, int64_t nwg) {
  constexpr int RING = 8 * 32 * D * 2, LDS = JOINT && KS == 1 ? RING : PrefixLds<D>::bytes;
  static_assert(LDS >= RING, "both item kinds fit");
  __shared__ __align__(16) uint16_t smem[LDS / 2];
  __shared__ int seen[JOINT && KS > 1 ? 1 : 128];
  if constexpr (JOINT && KS > 1) {
    prefix_attend<T, D>(p, prefix_item(p, xcd_logical_id(blockIdx.x, nwg), true), smem);
  } else if constexpr (JOINT) {
    prefix_attend_pipe<T, D>(p, prefix_item(p, xcd_logical_id(blockIdx.x, nwg), true), reinterpret_cast<char *>(smem), seen);
  } else {
    const int64_t np = p.Hkv * p.plan.prefix_tiles * p.plan.prefix_runs;
    if ((int64_t)blockIdx.x < np)
      prefix_attend_pipe<T, D>(p, prefix_item(p, xcd_logical_id(blockIdx.x, np), true), reinterpret_cast<char *>(smem), seen);
    else
      prefix_attend<T, D>(p, prefix_item(p, (int64_t)blockIdx.x - np, false), smem);
  }
}

// ---- f32 on the bf16 matrix cores ------------------------------------------------
//
// attn_f32x3_kernel's arithmetic over two key ranges: q, k, v and the probabilities as three exact bf16 terms each, six
// significant products an MFMA step, scores, probabilities and sums in f32. 128 rows a workgroup, 32 a wavefront; blocks of
// 32 keys are loaded as f32 (zeros past the range), split in registers and stored as three bf16 planes each of K and V,
// double-buffered. A wavefront without rows only stages.
template <int D, bool JOINT, int MINW>
__global__ __launch_bounds__(256, MINW) void prefix_f32_kernel(PrefixParams p, int64_t nwg) {
  using op_t = bf16x8_t;
  using M = Mma<BF16>;
  constexpr int BK = 32, NC = D / 16, NDT = D / 32;
  constexpr int KROW = D + 8;              // bf16 per plane row
  constexpr int PL = BK * KROW;            // one plane of one block
  constexpr int KCH = BK * D / 4 / 256;    // 16-byte f32 chunks of K (and of V) per thread and block
  __shared__ __align__(16) uint16_t smem[2 * 6 * PL];  // [buffer][K planes 0..2, V planes 0..2]
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int64_t npi = JOINT ? nwg : p.Hkv * p.plan.prefix_tiles * p.plan.prefix_runs;
  const bool first = JOINT || (int64_t)blockIdx.x < npi;
  const PrefixItem w = prefix_item(p, first ? xcd_logical_id(blockIdx.x, npi) : (int64_t)blockIdx.x - npi, first);
  const int64_t g = w.r0 + wave * 32 + l32;
  const bool live = g < w.rlim, rows = w.r0 + wave * 32 < w.rlim;
  const int np = (int)((w.p1 - w.p0 + BK - 1) / BK), no = (int)((w.o1 - w.o0 + BK - 1) / BK), nkv = np + no;
  const int pn = (int)(w.p1 - w.p0), on = (int)(w.o1 - w.o0);

  op_t q[3][NC];
  int seen, all_seen;  // own keys from o0 on that this lane's row sees; that every row of the tile sees
  {
    const PrefixRow row = prefix_row(p, w.kv, live ? g : w.rlim - 1);
    const int64_t len = own_len(p, w.b);
    seen = (int)(own_seen(p, len, row.i) - w.o0);
    all_seen = __builtin_amdgcn_readfirstlane((int)(own_seen(p, len, (w.r0 - w.b * p.Lq * p.G) / p.G) - w.o0));
    const float *qr = reinterpret_cast<const float *>(p.q) + row.b * p.q_sb + row.h * p.q_sh + row.i * p.q_st;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float x[8];
      Chunk<F32>::load<false>(qr + c * 16 + 8 * hh, x);
      u32x4_t x1, x2, x3;
#pragma unroll
      for (int e = 0; e < 4; ++e) split3_into(x[2 * e], x[2 * e + 1], x1, x2, x3, e);
      q[0][c] = __builtin_bit_cast(op_t, x1);
      q[1][c] = __builtin_bit_cast(op_t, x2);
      q[2][c] = __builtin_bit_cast(op_t, x3);
    }
  }
  const float *pk = reinterpret_cast<const float *>(p.pk) + w.kv * p.pk_sh + w.p0 * p.pk_st;
  const float *pv = reinterpret_cast<const float *>(p.pv) + w.kv * p.pv_sh + w.p0 * p.pv_st;
  const float *ok = reinterpret_cast<const float *>(p.k) + w.b * p.k_sb + w.kv * p.k_sh + w.o0 * p.k_st;
  const float *ov = reinterpret_cast<const float *>(p.v) + w.b * p.v_sb + w.kv * p.v_sh + w.o0 * p.v_st;
  // staging: chunk t + 256 i holds floats 4 (c % (D / 4)) .. of the block's row c / (D / 4)
  float4 rk[KCH], rv[KCH];
  auto load = [&](int j) {
    const bool pre = j < np;
    const int at = (pre ? j : j - np) * BK, left = (pre ? pn : on) - at;
    const int64_t kst = pre ? p.pk_st : p.k_st, vst = pre ? p.pv_st : p.v_st;
    const float *kb = (pre ? pk : ok) + at * kst, *vb = (pre ? pv : ov) + at * vst;
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + i * 256, r = c / (D / 4), o = (c % (D / 4)) * 4;
      rk[i] = rv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < left) {
        rk[i] = *reinterpret_cast<const float4 *>(kb + r * kst + o);
        rv[i] = *reinterpret_cast<const float4 *>(vb + r * vst + o);
      }
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + i * 256, off = c / (D / 4) * KROW + (c % (D / 4)) * 4;
      const Split3 ka = split3_bf16(rk[i].x, rk[i].y), kb = split3_bf16(rk[i].z, rk[i].w);
      const Split3 va = split3_bf16(rv[i].x, rv[i].y), vb = split3_bf16(rv[i].z, rv[i].w);
      uint16_t *d = smem + buf * 6 * PL + off;
      *reinterpret_cast<uint2 *>(d) = make_uint2(ka.t1, kb.t1);
      *reinterpret_cast<uint2 *>(d + PL) = make_uint2(ka.t2, kb.t2);
      *reinterpret_cast<uint2 *>(d + 2 * PL) = make_uint2(ka.t3, kb.t3);
      *reinterpret_cast<uint2 *>(d + 3 * PL) = make_uint2(va.t1, vb.t1);
      *reinterpret_cast<uint2 *>(d + 4 * PL) = make_uint2(va.t2, vb.t2);
      *reinterpret_cast<uint2 *>(d + 5 * PL) = make_uint2(va.t3, vb.t3);
    }
  };
  f32x16_t o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = f32x16_t{};
  float m = -3e38f, l = 0.f;
  const float c2 = p.scale * kLog2e;
  typedef short s16x4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
  auto compute = [&](int j) {
    const uint16_t *K1 = smem + (j & 1) * 6 * PL, *V1 = K1 + 3 * PL;
    f32x16_t s = f32x16_t{};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int off = l32 * KROW + (2 * c + hh) * 8;
      const op_t a1 = *reinterpret_cast<const op_t *>(K1 + off), a2 = *reinterpret_cast<const op_t *>(K1 + PL + off);
      const op_t a3 = *reinterpret_cast<const op_t *>(K1 + 2 * PL + off);
      s = M::run(a3, q[0][c], s);
      s = M::run(a2, q[1][c], s);
      s = M::run(a1, q[2][c], s);
      s = M::run(a2, q[0][c], s);
      s = M::run(a1, q[1][c], s);
      s = M::run(a1, q[0][c], s);
    }
    // this lane's row sees keys below lim of the block; lane holds keys 8 (i / 4) + 4 hh + i % 4
    if (j < np ? (j + 1) * BK > pn : (j - np + 1) * BK > all_seen) {
      const int lim = (j < np ? pn - j * BK : seen - (j - np) * BK) - 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i >> 2) + (i & 3) >= lim) s[i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
    const float cand = half_swap_max(mx) * c2;
    const float mn = cand > m + 8.f ? cand : m;
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    float ls = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c2, -mn));
      ls += s[i];
    }
    l = l * alpha + ls;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
    }
    // V^T fragments of each plane: see attn_mfma_kernel
    auto vfrag = [&](int pl, int dt, int jj) {
      const int g16 = lane & 15;
      const int vrow = 16 * jj + 4 * hh + (g16 >> 2), vcol = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (g16 & 3);
      const uint16_t *vr = V1 + pl * PL + vrow * KROW + vcol;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vr));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vr + 8 * KROW));
      return __builtin_bit_cast(op_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      u32x4_t x1, x2, x3;
#pragma unroll
      for (int e = 0; e < 4; ++e) split3_into(s[8 * jj + 2 * e], s[8 * jj + 2 * e + 1], x1, x2, x3, e);
      const op_t P1 = __builtin_bit_cast(op_t, x1), P2 = __builtin_bit_cast(op_t, x2), P3 = __builtin_bit_cast(op_t, x3);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const op_t v1 = vfrag(0, dt, jj), v2 = vfrag(1, dt, jj), v3 = vfrag(2, dt, jj);
        o[dt] = M::run(v3, P1, o[dt]);
        o[dt] = M::run(v2, P2, o[dt]);
        o[dt] = M::run(v1, P3, o[dt]);
        o[dt] = M::run(v2, P1, o[dt]);
        o[dt] = M::run(v1, P2, o[dt]);
        o[dt] = M::run(v1, P1, o[dt]);
      }
    }
  };
  if (nkv > 0) {
    load(0);
    store(0);
    lds_barrier();
    for (int j = 0; j < nkv; ++j) {
      if (j + 1 < nkv) load(j + 1);
      if (rows) compute(j);
      if (j + 1 < nkv) store((j + 1) & 1);
      lds_barrier();
    }
  }
  const float total = half_swap_sum(l);
  if (!live) return;
  // lane holds dims dt * 32 + 8 g4 + 4 hh + {0..3}
  float *dst;
  float f = 1.f;
  if (p.plan.parts > 1) {
    const int64_t per = p.B * p.Lq * p.G, all = per * p.Hkv, r = w.part * all + w.kv * per + g;
    const bool none = total == 0.f;
    if (hh == 0) *reinterpret_cast<float2 *>(p.ws + p.plan.parts * all * D + r * 2) = make_float2(none ? -INFINITY : m, total);
    if (none) return;
    dst = p.ws + r * D;
  } else {
    const PrefixRow row = prefix_row(p, w.kv, g);
    dst = reinterpret_cast<float *>(p.o) + row.b * p.o_sb + row.h * p.o_sh + row.i * p.o_st;
    f = total == 0.f ? 0.f : 1.f / total;
  }
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<float4 *>(dst + dt * 32 + 8 * g4 + 4 * hh) =
          make_float4(o[dt][4 * g4] * f, o[dt][4 * g4 + 1] * f, o[dt][4 * g4 + 2] * f, o[dt][4 * g4 + 3] * f);
}

// Merges a row's partial results: M = max m_s, out = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M). D / 4 lanes hold a row, 16
// bytes each; GP groups of them take every GP th part, U loads in flight, and their results are added in group order
// through LDS. A part that saw no key (m = -inf) has left no O: its weight is zero and what was read for it is dropped.
template <typename T, int D, int GP, int U>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixParams p) {
  constexpr int LPR = D / 4, RPB = 256 / (LPR * GP);
  __shared__ float4 so[GP > 1 ? 256 : 1];
  __shared__ float2 sml[GP > 1 ? 256 : 1];
  const int64_t per = p.B * p.Lq * p.G, rows = per * p.Hkv;
  const int t = threadIdx.x, grp = t / LPR % GP;
  int64_t r = (int64_t)blockIdx.x * RPB + t / (LPR * GP);
  const bool live = r < rows;
  r = live ? r : rows - 1;
  const int d = (t % LPR) * 4;
  const float2 *ml = reinterpret_cast<const float2 *>(p.ws + p.plan.parts * rows * D);
  const int parts = (int)p.plan.parts;
  float m = -INFINITY, l = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float mp, float lp, const float4 &x) {
    const float mn = fmaxf(m, mp), mb = mn == -INFINITY ? 0.f : mn;
    const float a = __builtin_amdgcn_exp2f(m - mb), b = __builtin_amdgcn_exp2f(mp - mb);
    const bool none = mp == -INFINITY;
    m = mn;
    l = l * a + lp * b;
    acc[0] = acc[0] * a + (none ? 0.f : x.x * b);
    acc[1] = acc[1] * a + (none ? 0.f : x.y * b);
    acc[2] = acc[2] * a + (none ? 0.f : x.z * b);
    acc[3] = acc[3] * a + (none ? 0.f : x.w * b);
  };
  for (int s0 = grp; s0 < parts; s0 += GP * U) {
    float2 v[U];
    float4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * GP < parts ? s0 + u * GP : s0;
      v[u] = ml[s * rows + r];
      x[u] = *reinterpret_cast<const float4 *>(p.ws + (s * rows + r) * D + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * GP < parts) add(v[u].x, v[u].y, x[u]);
  }
  if constexpr (GP > 1) {
    so[t] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    sml[t] = make_float2(m, l);
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int g = 1; g < GP; ++g) add(sml[t + g * LPR].x, sml[t + g * LPR].y, so[t + g * LPR]);
  }
  if (!live) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t kv = r / per;
  const PrefixRow row = prefix_row(p, kv, r - kv * per);
  char *orow = reinterpret_cast<char *>(p.o) + (row.b * p.o_sb + row.h * p.o_sh + row.i * p.o_st + d) * T::bytes;
  if constexpr (T::bytes == 4) {
    *reinterpret_cast<float4 *>(orow) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
  } else {
    *reinterpret_cast<uint2 *>(orow) = make_uint2(Mma<T>::pack(acc[0] * inv, acc[1] * inv), Mma<T>::pack(acc[2] * inv, acc[3] * inv));
  }
}

// The other head dims up to 512 and unaligned rows, each type: one wavefront per row, f32 throughout; lanes over keys for the scores,
// over dims for the output. DPL: dims per lane.
__device__ __forceinline__ float wave_max_xor(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}
template <typename T, int DPL>
__global__ __launch_bounds__(256) void prefix_generic_kernel(PrefixParams p, int64_t rows) {
  constexpr int EB = T::bytes;
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;  // whole wavefronts leave; no barrier below
  const int64_t per = p.B * p.Lq * p.G, kv = r / per;
  const PrefixRow row = prefix_row(p, kv, r - kv * per);
  const char *qrow = reinterpret_cast<const char *>(p.q) + (row.b * p.q_sb + row.h * p.q_sh + row.i * p.q_st) * EB;
  const int64_t D = p.D;
  float qv[DPL], o[DPL];
#pragma unroll
  for (int u = 0; u < DPL; ++u) {
    const int64_t d = lane + 64 * u;
    qv[u] = d < D ? load1<T>(qrow, d) : 0.f;
    o[u] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto keys = [&](const char *kb, int64_t kst, const char *vb, int64_t vst, int64_t n) {
    for (int64_t j0 = 0; j0 < n; j0 += 64) {
      const int64_t key = j0 + lane;
      const bool valid = key < n;
      const char *kr = kb + (valid ? key : n - 1) * kst * EB;
      float s = 0.f;
#pragma unroll
      for (int u = 0; u < DPL; ++u)
        for (int e = 0; e < 64; ++e) {
          const int64_t d = 64 * u + e;
          if (d >= D) break;
          s += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(qv[u]), e)) * load1<T>(kr, d);
        }
      s = valid ? s * p.scale : -INFINITY;
      const float mn = fmaxf(m, wave_max_xor(s));
      const float mb = mn == -INFINITY ? 0.f : mn;
      const float alpha = __expf(m - mb);
      const float pj = valid ? __expf(s - mb) : 0.f;
      l = l * alpha + wave_sum(pj);
      m = mn;
#pragma unroll
      for (int u = 0; u < DPL; ++u) o[u] *= alpha;
      const int nk = (int)(n - j0 < 64 ? n - j0 : 64);
      for (int kk = 0; kk < nk; ++kk) {
        const float pk = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(pj), kk));
        const char *vr = vb + (j0 + kk) * vst * EB;
#pragma unroll
        for (int u = 0; u < DPL; ++u) {
          const int64_t d = lane + 64 * u;
          if (d < D) o[u] += pk * load1<T>(vr, d);
        }
      }
    }
  };
  keys(reinterpret_cast<const char *>(p.pk) + kv * p.pk_sh * EB, p.pk_st,
       reinterpret_cast<const char *>(p.pv) + kv * p.pv_sh * EB, p.pv_st, p.P);
  keys(reinterpret_cast<const char *>(p.k) + (row.b * p.k_sb + kv * p.k_sh) * EB, p.k_st,
       reinterpret_cast<const char *>(p.v) + (row.b * p.v_sb + kv * p.v_sh) * EB, p.v_st,
       uniform(own_seen(p, own_len(p, row.b), row.i)));
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char *orow = reinterpret_cast<char *>(p.o) + (row.b * p.o_sb + row.h * p.o_sh + row.i * p.o_st) * EB;
#pragma unroll
  for (int u = 0; u < DPL; ++u) {
    const int64_t d = lane + 64 * u;
    if (d < D) store1<T>(orow, d, o[u] * inv);
  }
}

template <typename T>
hipError_t launch_prefix_generic(const PrefixParams &p, hipStream_t s) {
  const int64_t rows = p.B * p.H * p.Lq, groups = (rows + 3) / 4;
  if (groups > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)groups), block(256);
  if (p.D <= 64) hipLaunchKernelGGL((prefix_generic_kernel<T, 1>), grid, block, 0, s, p, rows);
  else if (p.D <= 128) hipLaunchKernelGGL((prefix_generic_kernel<T, 2>), grid, block, 0, s, p, rows);
  else if (p.D <= 256) hipLaunchKernelGGL((prefix_generic_kernel<T, 4>), grid, block, 0, s, p, rows);
  else hipLaunchKernelGGL((prefix_generic_kernel<T, 8>), grid, block, 0, s, p, rows);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_prefix_mfma(const PrefixParams &p, hipStream_t s) {
  const int64_t nwg = p.plan.wgs, rows = p.B * p.H * p.Lq;
  constexpr int LPR = D / 4;
  if (nwg > INT32_MAX || rows > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)nwg), block(256);
  if constexpr (T::code == LUX3D_F32) {
    constexpr int MINW = D == 64 ? 2 : 1;
    if (!p.plan.joint) hipLaunchKernelGGL((prefix_f32_kernel<D, false, MINW>), grid, block, 0, s, p, nwg);
    else hipLaunchKernelGGL((prefix_f32_kernel<D, true, MINW>), grid, block, 0, s, p, nwg);
  } else {
    constexpr int MINW = D == 64 ? 3 : 2;
    if (!p.plan.joint) hipLaunchKernelGGL((prefix_attn_kernel<T, D, false, 1, MINW>), grid, block, 0, s, p, nwg);
    else if (p.plan.ks == 2) hipLaunchKernelGGL((prefix_attn_kernel<T, D, true, 2, MINW>), grid, block, 0, s, p, nwg);
    else hipLaunchKernelGGL((prefix_attn_kernel<T, D, true, 1, MINW>), grid, block, 0, s, p, nwg);
  }
  if (hipError_t e = hipGetLastError()) return e;
  if (p.plan.parts > 1) {
    auto grid_of = [&](int gp) { return dim3((unsigned)((rows * LPR * gp + 255) / 256)); };
    const int groups = prefix_merge_groups(p.plan.parts, rows);
    if (groups == 0) hipLaunchKernelGGL((prefix_merge_kernel<T, D, 256 / LPR, 4>), grid_of(256 / LPR), block, 0, s, p);
    else if (groups == 4) hipLaunchKernelGGL((prefix_merge_kernel<T, D, 4, 4>), grid_of(4), block, 0, s, p);
    else hipLaunchKernelGGL((prefix_merge_kernel<T, D, 1, 8>), grid_of(1), block, 0, s, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_prefix_attention(int dt, const PrefixParams &p, hipStream_t s) {
  if (p.B <= 0 || p.H <= 0 || p.Lq <= 0) return hipSuccess;
  if (p.D < 1 || p.D > 512 || p.B * p.Lq * p.G > INT32_MAX) return hipErrorInvalidValue;
  switch (dt) {
    case LUX3D_BF16:
      if (p.mfma) return p.D == 64 ? launch_prefix_mfma<BF16, 64>(p, s) : launch_prefix_mfma<BF16, 128>(p, s);
      return launch_prefix_generic<BF16>(p, s);
    case LUX3D_F16:
      if (p.mfma) return p.D == 64 ? launch_prefix_mfma<F16, 64>(p, s) : launch_prefix_mfma<F16, 128>(p, s);
      return launch_prefix_generic<F16>(p, s);
    case LUX3D_F32:
      if (p.mfma) return p.D == 64 ? launch_prefix_mfma<F32, 64>(p, s) : launch_prefix_mfma<F32, 128>(p, s);
      return launch_prefix_generic<F32>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lux3d
