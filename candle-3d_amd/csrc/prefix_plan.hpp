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

inline PrefixPlan prefix_plan(int64_t B, int64_t H, int64_t Hkv, int64_t Lq, int64_t P, int64_t Ls) {
  PrefixPlan s;
  const int64_t rows = Lq * (H / Hkv);                                    // of one sequence and key head
  const int64_t pb = prefix_ceil(P, kPrefixKeys), ob = prefix_ceil(Ls, kPrefixKeys);
  const int64_t slots = 512;                                              // two workgroups on each of 256 CUs
  s.joint = rows >= 128 || B == 1;
  if (s.joint) {
    s.ks = rows > 64 ? 1 : 2;
    s.tile = 128 / s.ks;
    s.own_tiles = prefix_ceil(rows, s.tile);
    const int64_t tiles = B * Hkv * s.own_tiles, blocks = pb + ob;
    // too few tiles for the chip: runs of the keys that fill it once, four blocks or more each
    int64_t runs = slots / tiles;
    if (runs > blocks / 4) runs = blocks / 4;
    s.own_run = runs > 1 ? prefix_ceil(blocks, runs) : blocks > 0 ? blocks : 1;
    s.own_runs = blocks > 0 ? prefix_ceil(blocks, s.own_run) : 1;
    s.parts = s.own_runs;
    s.wgs = tiles * s.own_runs;
    return s;
  }
  s.prefix_tiles = prefix_ceil(B * rows, s.tile);
  s.own_tiles = prefix_ceil(rows, s.own_tile);
  // the prefix fills the chip once, beside the own keys' workgroups
  const int64_t tiles = Hkv * s.prefix_tiles, own = Hkv * B * s.own_tiles;
  int64_t runs = prefix_ceil(slots / 2, tiles);
  if (runs > pb / 2) runs = pb / 2;
  s.prefix_run = runs > 1 ? prefix_ceil(pb, runs) : pb > 0 ? pb : 1;
  runs = prefix_ceil(slots, own);
  if (runs > ob / 4) runs = ob / 4;
  s.own_run = runs > 1 ? prefix_ceil(ob, runs) : ob > 0 ? ob : 1;
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

}  // namespace lux3d
