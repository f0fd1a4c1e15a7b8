// mxfp4_tiles.hpp -- which kernel and tile a linear on microscaled 4-bit weights
// takes: the measured costs and the choice among them, host code without HIP.
#pragma once
#include <cmath>
#include <cstdint>

namespace lux3d {

// How x enters: packed (on the scaled matrix instructions), 2-byte values, f32.
enum MxKind : int { MX_PACKED = 0, MX_2BYTE = 1, MX_F32 = 2 };

// rows x cols of y and of the weights' rows (gated: half of cols outputs), the
// stages of k shared by `groups` groups of wavefronts. 256 x 256 of packed x:
// workgroups that stay for several tiles.
struct MxTileId {
  int rows, cols, groups;
};

// The rows below `rows` in tiles of `tile`, the rest (16 at most) as few rows in
// the same launch; rows 0: the few-rows kernel takes all.
struct MxChoice {
  MxTileId tile;
  int64_t rows;
};

inline double mx_up(int64_t a, int64_t b) { return (double)((a + b - 1) / b); }

// Weight tiles of 16 rows that a workgroup of the few-rows kernel takes for up to
// 16 rows of x, which is read, and quantised or split into its terms, once for all
// of them: more than one where enough workgroups are left. us with 1 / 2 / 4, 1
// and 16 rows:
//   bf16 2048 -> 8192    4.4 / 4.2 / 7.0 and 7.7 / 6.6 / 9.5
//        4096 -> 16384  12.2 / 10.2 / 11.6 and 22.3 / 15.9 / 14.5
//        4096 -> 32000  20.1 / 16.9 / 15.7 and 40.4 / 27.4 / 22.1
//   f32  4096 -> 16384  19.1 / 14.8 / 14.6 and 37.1 / 23.6 / 19.2
//   x in 4 bits, bf16 4096 -> 16384  11.8 / 10.6 / 9.3 and 21.9 / 15.6 / 13.1
//   bf16 8192 -> 2048    6.9 / 9.2 / 13.3 and 12.6 / 16.2 / 21.6
//   gated bf16 1536 -> 9216   7.1 / 8.4 / 10.5 and 10.5 / 12.5 / 13.7
//              4096 -> 16384 17.2 / 15.4 / 19.2 and 27.1 / 21.9 / 22.7
inline int mx_few_tiles(bool plain_2byte, int64_t n, int64_t k, bool gated) {
  if (gated) return n >= 16384 && k >= 1024 ? 2 : 1;
  if (n < 8192 || k < 512) return 1;
  return k >= 1024 && n >= (plain_2byte ? 24576 : 16384) ? 4 : 2;
}

// The few-rows kernel's workgroup: row tiles of x and weight tiles of 16 rows each, wavefronts that share k.
struct MxFewTile {
  int rows, cols, waves;
};

// us with 4 / 8 / 16 wavefronts: 1 row, 8192 -> 2048 bf16 12.9 / 8.9 / 7.4, f32 19.3 / 13.8 / 11.0; 2048 -> 8192 4.5 / 4.5 /
// 4.5, f32 6.8 / 6.4 / 6.9; 1536 -> 9216 5.1 / 4.8 / 5.3; 33 rows, 8192 -> 2048 23.6 / 20.4 / 20.2, 1536 -> 9216 13.6 / 13.0 /
// 14.1. Four row tiles instead of two: 64 rows, 8192 -> 2048 20.7 -> 35.6, 2048 -> 8192 19.9 -> 19.6. Two groups in flight a
// wavefront: within 8%.
inline MxFewTile mx_few_tile(bool plain_2byte, int64_t m, int64_t n, int64_t k, bool gated) {
  if (m > 16) return {2, 1, 8};
  const int tiles = mx_few_tiles(plain_2byte, n, k, gated);
  return {1, tiles, tiles == 1 && k >= 6144 ? 16 : 8};
}

// Us of the few-rows kernel: a launch, the chain of a wavefront's groups of 128
// of k, and the loads of weights and of x, by the rows of a workgroup's tile.
// Fitted to 48, 24 and 24 sizes of up to 16 rows and 150 to 168 of more, within
// 8 to 16% (root mean square).
inline double mx_few_cost(MxKind kind, int64_t m, int64_t n, int64_t k, bool gated) {
  constexpr double f[3][2][5] = {
      // launch, chain, weights, x's rows, workgroup: up to 16 rows; more
      {{1.5, 1.12, 0.019, 0.0081, 0.0}, {2.0, 0.64, 0.048, 0.0003, 0.51}},
      {{1.5, 1.12, 0.036, 0.0076, 0.0}, {1.7, 1.39, 0.043, 0.0038, 0.46}},
      {{1.2, 1.99, 0.028, 0.0139, 0.0}, {1.2, 2.53, 0.0, 0.0111, 0.84}}};
  const bool few = m <= 16;
  const double *c = f[kind][few ? 0 : 1];
  const int64_t t = few ? 16 : 32;
  const double g = mx_up(k, 128), w = mx_up(n, 16) * mx_up(m, t) / 256;
  const double rows = (double)(m < t ? m : t) / (few ? mx_few_tiles(kind == MX_2BYTE, n, k, gated) : 1);
  return c[0] + c[1] * std::ceil(g / (few && k >= 6144 ? 16 : 8)) * (gated ? 1.41 : 1) + w * (g * (c[2] * (gated ? 2 : 1) + c[3] * rows) + c[4]);
}

// Us of the tiles: c + r (a stages + b). A workgroup alone on its CU takes a
// stages + b; w tiles a CU take r = s (th ceil(w) + (1 - th) w) times that, 1 at
// least: s below 1 where several share a CU, th what of a last round is idle.
// Fitted to 70 to 320 sizes each (k 128 to 8192, 17 to 16392 rows), within 4 to
// 16% where a tile is near the best (the 256 x 256 tile of packed x 22%). Of 1180
// sizes timed with every tile, the tile so chosen takes 1.0% (packed), 1.6% (2
// bytes) and 0.3% (f32) longer than the shortest on average. Of 624 sizes of 17 to
// 600 rows, few rows among the forms, it takes 0.9% longer, and 20 to 43% in eight:
// few rows where a tile is shorter (us; 160 rows of 4096 -> 1024 packed 9.5 against
// 6.7, bf16 19.4 against 13.6, gated 22.3 against 17.1; gated, 64 rows of 256 -> 5000
// bf16 7.3 against 5.6, of 1024 -> 4096 packed 6.2 against 5.0, 100 of 1536 -> 1536
// packed 7.1 against 5.9), and two rows past a tile apart (130 of 4096 -> 16384 packed
// 16.5 against 13.6, gated 32.5 against 24.2). Beside those: gated packed x of 48 rows
// of 8192 -> 2048 (with its quantisation 19.0 against few rows' 15.6), and 128 x 256
// tiles of short k (256 -> 5000 of 4098 rows 29.8 against 64 x 128's 25.8).
struct MxCost {
  MxTileId tile;
  double c, a, b, s, th;
  bool beside;  // two workgroups fit a CU's LDS
};

inline MxChoice mx_choose(MxKind kind, int64_t m, int64_t n, int64_t k, bool gated) {
  constexpr MxCost packed[] = {{{64, 64, 1}, 2.76, 0.142, 0.92, 0.88, 0.72, true},
                               {{64, 64, 2}, 1.99, 0.240, 2.16, 0.90, 1.00, true},
                               {{64, 128, 1}, 3.10, 0.190, 1.17, 1.04, 0.69, true},
                               {{128, 128, 1}, 2.97, 0.286, 2.82, 0.98, 0.80, true},
                               {{256, 256, 1}, 6.78, 0.595, 4.75, 1.35, 0.69, false}};
  constexpr MxCost two[] = {{{64, 64, 1}, 2.88, 0.257, 1.19, 0.68, 0.95, true},
                            {{64, 64, 2}, 1.71, 0.333, 3.00, 1.09, 0.89, false},
                            {{64, 64, 4}, 3.38, 0.576, 2.55, 1.24, 0.78, false},
                            {{64, 128, 1}, 3.34, 0.297, 1.33, 0.87, 0.64, true},
                            {{64, 128, 2}, 2.12, 0.453, 3.57, 1.07, 0.97, false},
                            {{64, 128, 4}, 4.14, 0.764, 3.58, 1.27, 0.75, false},
                            {{128, 128, 1}, 3.13, 0.419, 2.75, 0.98, 0.59, true},
                            {{128, 256, 1}, 5.45, 0.705, 3.89, 1.03, 0.65, true},
                            {{256, 256, 1}, 2.42, 1.070, 9.59, 1.21, 0.77, false}};
  constexpr MxCost f32[] = {{{64, 64, 4}, 2.83, 1.011, 3.83, 1.08, 0.92, false},
                            {{64, 128, 2}, 3.77, 0.666, 3.00, 0.91, 0.72, true},
                            {{64, 128, 4}, 3.78, 1.083, 5.16, 1.17, 0.86, false}};
  const MxCost *costs = kind == MX_PACKED ? packed : kind == MX_2BYTE ? two : f32;
  const int count = kind == MX_PACKED ? 5 : kind == MX_2BYTE ? 9 : 3;
  const int64_t depth = kind == MX_PACKED ? 128 : kind == MX_2BYTE ? 64 : 32;
  MxChoice best = {{16, 16, 1}, 0};
  if (m <= 16) return best;
  double least = mx_few_cost(kind, m, n, k, gated);
  for (int i = 0; i < count; ++i) {
    const MxCost &t = costs[i];
    if (gated && t.tile.cols == 64) continue;                                   // a gate's half of 32 columns
    if (kind == MX_PACKED && t.tile.rows == 256 && k < 512) continue;           // four stages a tile at least
    const double one = t.a * std::ceil(mx_up(k, depth) / t.tile.groups) + t.b;
    const double cols = mx_up(n, gated ? t.tile.cols / 2 : t.tile.cols);
    auto cost = [&](int64_t rows) {
      const double w = mx_up(rows, t.tile.rows) * cols / 256;
      return t.c + (w <= 1 ? 1 : std::fmax(1, t.s * (t.th * std::ceil(w) + (1 - t.th) * w))) * one;
    };
    const double whole = cost(m);
    if (whole < least) {
      least = whole;
      best = {t.tile, m};
    }
    // Few rows past the last whole tile (2 x 2049 tokens) as few rows, where that saves a row of tiles. Beside the tiles they
    // cost a tenth to two thirds of their own launch (1029 rows against 1024, us: f32 1024 -> 4096 28.4 / 27.5, gated f16
    // 23.8 / 21.0, 4098 against 4096, 1024 -> 4096 bf16 35.0 / 33.4), behind them, where no second workgroup fits a CU, all of it.
    const int64_t rest = m % t.tile.rows;
    if (rest >= 1 && rest <= 16 && m > t.tile.rows) {
      const double split = cost(m - rest) + (t.beside ? 0.4 : 1) * mx_few_cost(kind, rest, n, k, gated);
      if (split < least) {
        least = split;
        best = {t.tile, m - rest};
      }
    }
  }
  return best;
}

// Whether a call's rows lie close enough for the kernel of many rows: its descriptors span 256 rows of x and of the weights,
// and the scales of the whole matrix; its offsets, also into a tile of y, have 32 bits. ldx: elements between plain x's rows;
// xs_rows: rows of packed x's scales.
inline bool mx_gemm_fits(MxKind kind, int64_t ldx, int64_t xs_rows, int64_t n, int64_t k, int64_t ldy) {
  const int64_t lim = 0x7FFFFFFF, s = (k + 127) / 32;  // s: a row's scales, at most
  const int64_t xrow = kind == MX_PACKED ? k / 2 : ldx * (kind == MX_F32 ? 4 : 2) + 64;
  return 256 * xrow <= lim && 256 * k <= lim && 256 * 4 * ldy <= lim && s * n <= lim && (kind != MX_PACKED || s * xs_rows <= lim);
}

}  // namespace lux3d
