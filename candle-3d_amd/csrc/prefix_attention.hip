// prefix_attention.hip -- attention of a batch whose sequences share one long prefix of keys:
//   out[b, h, i] = softmax over the P prefix keys and the own keys j that query i sees of (q . k * scale), times v
// An own key j is seen when j < len_b and, with causality, j <= len_b - Lq + i. The prefix's K and V exist once, for all
// sequences; a head group of H / Hkv query heads shares a key head.
//
// What bounds it. Long queries: the matrix cores, 4 D operations a visible (query, key) pair. Decoding: the bytes of K
// and V. The rows that share a key head's prefix, of all sequences and of the group's heads, are therefore taken
// together, 64 rows a tile: the prefix is read once for up to 64 of them instead of once a row. Own keys are read by
// workgroups of their own. Every workgroup takes a run of key blocks, so that few rows still fill the chip, and leaves
// an unnormalised partial result (maximum, sum, O); a second kernel merges a row's partials in their order.
//
// Numerics: f32 scores, softmax with a running maximum and sums in f32. The 2-byte types' probabilities are rounded to
// the type for P v (the row sum adds the rounded ones), as lux3d_sdpa does; out is rounded once. A row that sees no key
// is zero.
//
// Masks. Keys past a sequence's length are never read: the buffer loads end at the last visible key and return zeros, so
// that a probability of zero meets a finite value. Inside a tile, keys that causality hides from some of its rows are
// read for the others; scores there become -inf whatever K holds, and V there is handled as described at `poison`.
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

__device__ __forceinline__ PrefixItem prefix_item(const PrefixParams &p, int64_t lid, int tile) {
  const PrefixPlan &s = p.plan;
  const int64_t R = p.Lq * p.G, run = s.run * kPrefixKeys;
  PrefixItem w;
  w.p0 = w.p1 = w.o0 = w.o1 = 0;
  if (s.joint) {
    // key heads outermost: the tiles of one XCD share a key head's prefix in its L2
    uint32_t x = (uint32_t)lid;
    const uint32_t tiles = (uint32_t)s.own_tiles, B = (uint32_t)p.B, runs = (uint32_t)s.own_runs;
    const uint32_t t = x % tiles;
    x /= tiles;
    w.b = x % B;
    x /= B;
    w.part = x % runs;
    w.kv = x / runs;
    w.r0 = w.b * R + (int64_t)t * tile;
    w.rlim = (w.b + 1) * R;
    // blocks of the prefix, then of the own keys, in runs
    const int64_t pb = (p.P + kPrefixKeys - 1) / kPrefixKeys;
    const int64_t j0 = w.part * s.run, j1 = j0 + s.run;
    w.p0 = j0 * kPrefixKeys;
    w.p1 = j1 * kPrefixKeys < p.P ? j1 * kPrefixKeys : p.P;
    w.o0 = j0 > pb ? (j0 - pb) * kPrefixKeys : 0;
    w.o1 = j1 > pb ? (j1 - pb) * kPrefixKeys : 0;
  } else {
    const uint32_t np = (uint32_t)(p.Hkv * s.prefix_tiles * s.prefix_runs);
    uint32_t x = (uint32_t)lid;
    if (x < np) {
      const uint32_t tiles = (uint32_t)s.prefix_tiles, runs = (uint32_t)s.prefix_runs;
      const uint32_t t = x % tiles;
      x /= tiles;
      w.part = x % runs;
      w.kv = x / runs;
      w.r0 = (int64_t)t * tile;
      w.rlim = p.B * R;
      w.b = 0;
      w.p0 = w.part * run;
      w.p1 = w.p0 + run < p.P ? w.p0 + run : p.P;
      return w;
    }
    x -= np;
    const uint32_t tiles = (uint32_t)s.own_tiles, runs = (uint32_t)s.own_runs, hkv = (uint32_t)p.Hkv;
    const uint32_t t = x % tiles;
    x /= tiles;
    const uint32_t pr = x % runs;
    x /= runs;
    w.kv = x % hkv;
    w.b = x / hkv;
    w.part = s.prefix_runs + pr;
    w.r0 = w.b * R + (int64_t)t * tile;
    w.rlim = (w.b + 1) * R;
    w.o0 = pr * run;
    w.o1 = w.o0 + run;
  }
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

// Matrix-core kernel of the 2-byte types. Four wavefronts: 4 / KS row groups of 32 rows, the KS wavefronts of a group
// taking every block's 64 / KS keys. S^T = K Q^T, O^T += V^T P^T as attn_mfma_kernel does it: each lane holds one row's
// scores of 16 keys, K and V blocks come by direct global -> LDS loads, two blocks deep.
template <typename T, int D, int KS, int MINW>
__global__ __launch_bounds__(256, MINW) void prefix_attn_kernel(PrefixParams p, int64_t nwg) {
  using M = Mma<T>;
  using op_t = typename M::op_t;
  constexpr int BKV = kPrefixKeys, NKT = BKV / 32 / KS, NDT = D / 32, TILE = 128 / KS;
  constexpr int KCH = BKV * D / 8 / 256;   // 16-byte chunks of K (and V) per thread and block
  constexpr int BUF = BKV * D;             // 2-byte elements of a block
  constexpr bool VEARLY = D == 128 && KS == 2;  // 128 rows leave no registers for it
  // the ring of two K and two V blocks; at the end the key groups' partial results
  constexpr int PW = KS > 1 ? (NDT * 16 + 2) * 64 : 0;  // floats of a wavefront
  constexpr int LDS = 4 * BUF * 2 > 4 * PW * 4 ? 4 * BUF * 2 : 4 * PW * 4;
  __shared__ __align__(16) uint16_t smem[LDS / 2];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int qg = wave / KS, kg = wave % KS, kt0 = kg * NKT;

  const PrefixItem w = prefix_item(p, xcd_logical_id(blockIdx.x, nwg), TILE);
  const int64_t g = w.r0 + qg * 32 + l32;          // this lane's row
  const bool live = g < w.rlim;
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
    const uint16_t *Ks = smem + buf * BUF, *Vs = smem + 2 * BUF + buf * BUF;
    f32x16_t s[NKT];
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt) {
      s[kt] = f32x16_t{};
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const int krow = (kt0 + kt) * 32 + l32;
        const op_t a = *reinterpret_cast<const op_t *>(Ks + krow * D + ((2 * c + hh) ^ k_swz<D>(krow)) * 8);
        s[kt] = M::run(a, qf[c], s[kt]);
      }
    }
    // this lane's row sees keys below lim of the block; lane holds keys 8 (i / 4) + 4 hh + i % 4 of each 32-key tile
    int lim = BKV;
    if constexpr (MASK) {
      lim = j < np ? (int)(w.p1 - w.p0) - j * BKV : seen - (int)w.o0 - (j - np) * BKV;
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((kt0 + kt) * 32 + 8 * (i >> 2) + (i & 3) >= lim - 4 * hh) s[kt][i] = -INFINITY;
    }
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
    // V^T fragment of dim tile dt, keys 16 jj ..: see attn_mfma_kernel
    auto vfrag = [&](int dt, int kt, int jj) {
      const int g16 = lane & 15;
      const int vrow = (kt0 + kt) * 32 + 16 * jj + 4 * hh + (g16 >> 2);
      const int vcol = dt * 32 + 16 * ((lane >> 4) & 1) + 4 * (g16 & 3);
      const uint16_t *vr = Vs + vrow * D + ((vcol >> 3) ^ v_swz<D>(vrow)) * 8 + (vcol & 7);
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vr));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(vr + 8 * D));
      return __builtin_bit_cast(op_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    // V's fragments are read before the softmax, which hides their latency
    op_t vf[VEARLY ? NDT * NKT * 2 : 1];
    if constexpr (VEARLY) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) vf[(dt * NKT + kt) * 2 + jj] = vfrag(dt, kt, jj);
      __builtin_amdgcn_sched_barrier(0);
    }

    // running maximum: it moves when a block's exceeds it by 2^8, so that most blocks need no rescale
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kt][i]);
    const float cand = half_swap_max(mx) * c2;
    const float mn = cand > m + 8.f ? cand : m;
    const float mb = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every probability is exp2(-inf)
    const float alpha = __builtin_amdgcn_exp2f(m - mb);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] *= alpha;
    }
    m = mn;
    op_t pf[NKT * 2];
    float ls = 0.f;
#pragma unroll
    for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        u32x4_t pk4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][8 * jj + 2 * e], c2, -mb));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][8 * jj + 2 * e + 1], c2, -mb));
          pk4[e] = M::pack(p0, p1);
          ls = M::sum2(pk4[e], ls);
        }
        pf[kt * 2 + jj] = __builtin_bit_cast(op_t, pk4);
      }
    l = l * alpha + ls;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int kt = 0; kt < NKT; ++kt)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
          o[dt] = M::run(VEARLY ? vf[(dt * NKT + kt) * 2 + jj] : vfrag(dt, kt, jj), pf[kt * 2 + jj], o[dt]);
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

  if constexpr (KS > 1) {
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
  }

  const float total = half_swap_sum(l);
  if (!live) return;
  // lane holds dims dt * 32 + 8 g4 + 4 hh + {0..3}, g4 = 0..3
  if (p.plan.parts > 1) {
    const int64_t rows = p.B * p.Lq * p.G * p.Hkv, r = (w.part * p.Hkv + w.kv) * (p.B * p.Lq * p.G) + g;
    float *po = p.ws + r * D;
    if (kg == 0 && hh == 0) *reinterpret_cast<float2 *>(p.ws + p.plan.parts * rows * D + r * 2) = make_float2(m, total);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      if (KS > 1 && dt % KS != kg) continue;
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
    if (KS > 1 && dt % KS != kg) continue;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4)
      *reinterpret_cast<uint2 *>(orow + (dt * 32 + 8 * g4 + 4 * hh) * 2) =
          make_uint2(M::pack(o[dt][4 * g4] * inv, o[dt][4 * g4 + 1] * inv),
                     M::pack(o[dt][4 * g4 + 2] * inv, o[dt][4 * g4 + 3] * inv));
  }
}

// Merges a row's partial results in their order: M = max m_s, out = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M). D / 4
// lanes a row, 16 bytes each. A part that saw no key (m = -inf) is not read.
template <typename T, int D>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixParams p) {
  constexpr int LPR = D / 4, RPB = 256 / LPR;
  const int64_t per = p.B * p.Lq * p.G, rows = per * p.Hkv;
  const int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR;
  if (r >= rows) return;
  const int d = (int)(threadIdx.x % LPR) * 4;
  const float2 *ml = reinterpret_cast<const float2 *>(p.ws + p.plan.parts * rows * D);
  float m = -INFINITY, l = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t s = 0; s < p.plan.parts; ++s) {
    const float2 v = ml[s * rows + r];
    if (v.x == -INFINITY) continue;
    const float4 x = *reinterpret_cast<const float4 *>(p.ws + (s * rows + r) * D + d);
    const float mn = fmaxf(m, v.x);
    const float a = __builtin_amdgcn_exp2f(m - mn), b = __builtin_amdgcn_exp2f(v.x - mn);
    m = mn;
    l = l * a + v.y * b;
    acc[0] = acc[0] * a + x.x * b;
    acc[1] = acc[1] * a + x.y * b;
    acc[2] = acc[2] * a + x.z * b;
    acc[3] = acc[3] * a + x.w * b;
  }
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

// Any head dim up to 512, any alignment, f32: one wavefront per row, f32 throughout; lanes over keys for the scores,
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
  const int64_t nwg = p.plan.wgs;
  if (nwg > INT32_MAX || p.B * p.Lq * p.G > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)nwg), block(256);
  constexpr int MINW = D == 64 ? 3 : 2;
  if (p.plan.ks == 1) hipLaunchKernelGGL((prefix_attn_kernel<T, D, 1, MINW>), grid, block, 0, s, p, nwg);
  else hipLaunchKernelGGL((prefix_attn_kernel<T, D, 2, MINW>), grid, block, 0, s, p, nwg);
  if (hipError_t e = hipGetLastError()) return e;
  if (p.plan.parts > 1) {
    const int64_t rows = p.B * p.H * p.Lq, per = 256 / (D / 4);
    hipLaunchKernelGGL((prefix_merge_kernel<T, D>), dim3((unsigned)((rows + per - 1) / per)), block, 0, s, p);
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
    case LUX3D_F32: return launch_prefix_generic<F32>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace lux3d
