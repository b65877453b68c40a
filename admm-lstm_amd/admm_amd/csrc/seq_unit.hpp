// seq_unit.hpp -- operands and work memory of the gated unit's kernels.
#pragma once
#include <stdint.h>

namespace seq {

constexpr int64_t kUnitMaxRows = 0x7fffffff - 255;   // row numbers up to the last tile's end are 32-bit integers

struct UnitArgs {
  int M, D, F, act, dtype;
  const void *x, *wg, *wu;
  int64_t x_ld, w_ld, wu_ld;
  bool copy_x, copy_w;          // operands that need padded copies (those held as planes: always)
  char *xp, *wgp, *wup;         // their copies
  int64_t D8, F8;               // row lengths of the copies, in elements
  float *pre;                   // a, then b [M, F] (NULL: not kept)
  void* y;
  // gradients
  const void* dy;
  int64_t dy_ld;
  char *dap, *dbp;              // [planes][M, F8]
  float *sums;                  // dWg and dWu in parts, where they are formed so (unit_parts)
  void *dx, *dwg, *dwu;
};

// Tile sizes of an m x n result (n: both projections' columns): 0: 256 x 256 (8 waves, one workgroup a compute unit), 1: 128 x
// 128 (4 waves, two), 2: 64 x 64 (4 waves, four), 3: 192 x 256 (8 waves, one; not where A is transposed on its way).  The one
// whose rounds over the 256 units take the least: a round is the work of a unit's workgroups over the share of the first one's
// rate that the tile reaches, from these times (us, D 2048, F 4096, bf16 and f32, tiles 0 to 3):
//   M 4096: 130, 139, 240, 148 and 695, 774, 1986, 780;  M 2048: 71, 87, 141, 99 and 383, 403, 801, 506;
//   M 1536 (a whole round of tile 3): 64, 61, 95, 54 and 330, 342, 576, 284.
// parts: of the inner axis; time: rounds of the first tile over the whole inner axis, times `parts`.
inline int tile_for(int64_t m, int64_t n, bool with3, int parts, double* time) {
  auto rounds = [](int64_t tiles, int slots) { return (double)((tiles + slots - 1) / slots); };
  auto count = [&](int r, int c) { return ((m + r - 1) / r) * ((n + c - 1) / c) * parts; };
  const double cost[4] = {rounds(count(256, 256), 256), rounds(count(128, 128), 512) * 2 / 4 / 0.9, rounds(count(64, 64), 1024) * 4 / 16 / 0.5,
                          rounds(count(192, 256), 256) * 3 / 4 / 0.98};
  int best = 0;
  for (int t = 1; t < (with3 ? 4 : 3); ++t) best = cost[t] < cost[best] ? t : best;
  if (time) *time = cost[best];
  return best;
}

// threads of a launch of such tiles, along its first axis
inline int64_t tile_threads(int tile, int64_t m, int64_t n) {
  constexpr int rows[4] = {256, 128, 64, 192}, cols[4] = {256, 128, 64, 256}, threads[4] = {512, 256, 256, 512};
  return (m + rows[tile] - 1) / rows[tile] * ((n + cols[tile] - 1) / cols[tile]) * threads[tile];
}

// dWg and dWu have few tiles where the layer is narrow, and sum over all M rows: the sums are formed in parts, which a second
// kernel adds up (in order), where that takes less time.  A round of 256 x 256 takes 30 ns a row (fp16: three times that, f32: six
// times), the parts are written and read at memory's rate, and another launch takes 5 us.  All gradients together, in us, and with one part:
//   f32: 262144 x 256 x 512: 2431 (19342), 65536 x 128 x 256: 351 (3723), 8192 x 512 x 1365: 621 (790), 1500 x 256 x 512: 102 (130);
//   fp16: 1404 (9751), 209 (1583), 331 (404), 63 (74);  bf16: 724 (3483), 111 (561), 174 (190), 61 (57).
struct UnitParts {
  int tile, parts;
};
inline UnitParts unit_parts(int64_t M, int D, int F, int dtype) {
  UnitParts best = {0, 1};
  double least = 0;
  for (int p = 1; p <= 64 && (p == 1 || M / p >= 512); p *= 2) {
    double rounds;
    const int tile = tile_for(D, 2 * (int64_t)F, false, p, &rounds);
    const double us = rounds / p * M * (dtype == SEQ_FP32 ? 0.18 : dtype == SEQ_FP16 ? 0.09 : 0.03) + (p > 1 ? 5 + p * 16e-6 * D * F / 5 : 0);
    if (p == 1 || us < least) best = {tile, p}, least = us;
  }
  return best;
}

}  // namespace seq
