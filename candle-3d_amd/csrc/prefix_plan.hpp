// prefix_plan.hpp -- how a shared-prefix attention is cut into workgroups: host code without HIP.
#pragma once
#include <cstdint>

namespace lux3d {

constexpr int kPrefixKeys = 64;  // keys of a block

// A query row is (sequence b, position i, query head of the key head's group): rows = B * Lq * group per key head,
// sequence-major, so that a tile of consecutive rows is one sequence's, or several sequences'.
//
// joint: a workgroup takes `tile` rows of one sequence through the prefix's and the sequence's own keys (long Lq).
// Otherwise the prefix is read once for `tile` rows of all sequences together, and each sequence's own keys by workgroups
// of their own, own_tile rows each: few rows (decoding). Key ranges are cut into runs of blocks, one workgroup each;
// `parts` partial results a row are merged by a second kernel (parts 1: the first writes out itself).
struct PrefixPlan {
  bool joint = true;
  int ks = 1;                 // joint: key groups of a workgroup's four wavefronts, 128 / ks rows a tile
  int tile = 128, own_tile = 64;
  int64_t prefix_tiles = 0, prefix_run = 1, prefix_runs = 0;
  int64_t own_tiles = 0, own_run = 1, own_runs = 0;  // joint: over the blocks of both
  int64_t parts = 1, wgs = 0;
};

inline int64_t prefix_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Joint: into how many runs the keys of `tiles` tiles of 128 rows are cut, by the time that follows: the busiest CU's
// blocks (us a block with 1, 2 or 3 workgroups on the CU: D 64 0.83, 1.25, 1.85, D 128 1.07, 1.9), and for more than one
// run the merge, 4 us and the partial results' bytes at 4 TB/s. us, one run / the one so chosen / the best of 1 to 16: 2 x
// 16 heads x 300 on 1029 + 300 24.7 / 20.6 / 20.6, 16 x 1374 on 10992 + 1374 165 / 98.9 / 98.9, 16 x 130 on 16000 + 130
// 211 / 31.3 / 31.3 (D 64); 3 x 12 / 4 x 333 on 4001 + 707 85.1 / 51.0 / 51.0, 12 x 1029 on 4000 + 1029 90.4 / 58.2 / 52.3,
// 4 x 12 x 200 on 1029 + 200 28.3 / 26.9 / 26.9, 2 x 12 x 2000 on 4000 + 2000 167 / 167 / 163 (D 128).
inline int64_t prefix_joint_runs(int64_t tiles, int64_t blocks, int64_t rows, int64_t D, bool f32) {
  const double t64[4] = {0, 0.83, 1.25, 1.85}, t128[3] = {0, 1.07, 1.9}, f64[3] = {0, 3.3, 5.0}, f128[2] = {0, 6.6};
  const int per_cu = (D <= 64 ? 3 : 2) - f32;
  const double *t = f32 ? (D <= 64 ? f64 : f128) : D <= 64 ? t64 : t128;
  int64_t best = 1;
  double least = 0;
  for (int64_t runs = 1; runs <= 16 && (runs == 1 || runs <= blocks / 2); ++runs) {
    const int64_t m = prefix_ceil(tiles * runs, 256);
    double us = (double)prefix_ceil(blocks, runs) * ((double)(m / per_cu) * t[per_cu] + t[m % per_cu]);
    if (runs > 1) us += 4 + (double)rows * (double)runs * (double)D * 8 / 4e6;
    if (runs == 1 || us < least) least = us, best = runs;
  }
  return best;
}

inline PrefixPlan prefix_plan(int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t P, int64_t Ls, int64_t D,
                              bool f32) {
  PrefixPlan s;
  const int64_t rows = Lq * (H / Hkv);                                    // of one sequence and key head
  const int64_t pb = prefix_ceil(P, kPrefixKeys), ob = prefix_ceil(Ls, kPrefixKeys);
  auto run_of = [](int64_t blocks, int64_t runs) { return blocks <= 0 ? 1 : runs > 1 ? prefix_ceil(blocks, runs) : blocks; };
  s.joint = rows >= 128 || B == 1;
  if (s.joint) {
    s.ks = rows > 64 || f32 ? 1 : 2;
    s.tile = 128 / s.ks;
    s.own_tiles = prefix_ceil(rows, s.tile);
    const int64_t tiles = B * Hkv * s.own_tiles, blocks = pb + ob;
    // few rows, bound by the keys' bytes: runs that fill the chip twice, two blocks or more each
    int64_t runs = rows > 64 ? prefix_joint_runs(tiles, blocks, B * H * Lq, D, f32) : 512 / tiles;
    if (runs > blocks / 2) runs = blocks / 2;
    s.own_run = run_of(blocks, runs);
    s.own_runs = blocks > 0 ? prefix_ceil(blocks, s.own_run) : 1;
    s.parts = s.own_runs;
    s.wgs = tiles * s.own_runs;
    return s;
  }
  if (f32) s.own_tile = 128;
  s.prefix_tiles = prefix_ceil(B * rows, s.tile);
  s.own_tiles = prefix_ceil(rows, s.own_tile);
  // The prefix's workgroups take half of the CUs, or all where there are few own keys: with more of them the own keys'
  // workgroups, which wait for memory, start late. us with 64 / 128 / 256 of them: 64 x 32 / 8 heads on 16384 + 1000 (D
  // 128) 80.7 / 50.5 / 59.6, 4 x 16 on 16384 + 2000 (D 64) 62.7 / 36.4 / 23.8, 64 x 16 on 4096 + 100 21.9 / 21.5 / 21.4.
  const int64_t tiles = Hkv * s.prefix_tiles, own = Hkv * B * s.own_tiles;
  int64_t runs = prefix_ceil(2 * own * ob <= tiles * pb ? 256 : 128, tiles);
  if (runs > pb / 2) runs = pb / 2;
  s.prefix_run = run_of(pb, runs);
  runs = prefix_ceil(512, own);
  if (runs > ob / 4) runs = ob / 4;
  s.own_run = run_of(ob, runs);
  s.prefix_runs = prefix_ceil(pb, s.prefix_run);
  s.own_runs = prefix_ceil(ob, s.own_run);
  s.parts = s.prefix_runs + s.own_runs;
  if (s.parts < 1) s.own_runs = s.parts = 1;
  s.wgs = tiles * s.prefix_runs + own * s.own_runs;
  return s;
}

// f32 values of workspace: the parts' unnormalised outputs and their (maximum, sum)
inline int64_t prefix_workspace(const PrefixPlan &s, int64_t B, int64_t H, int64_t Lq, int64_t D) {
  return s.parts > 1 ? s.parts * B * H * Lq * (D + 2) : 0;
}

// How many groups of lanes share a row's partial results in the merge: a row's lanes alone where few parts of many rows keep
// every lane busy, the whole workgroup (0) where a row has many.
inline int prefix_merge_groups(int64_t parts, int64_t rows) {
  return parts > 32 ? 0 : parts > 8 || rows < 4096 ? 4 : 1;
}

}  // namespace lux3d
