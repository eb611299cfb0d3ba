// Which kernel makes a product: plain arithmetic on the sizes, of the host.
//
// The kernel is the one whose estimated time is least, t = rounds of resident workgroups * (us per stage * stages + us per
// round), a stage 128 bytes of the contraction (8 bits: a block of k), with the rates that each was measured at.  A round is
// what `cus` CUs hold at a time (c2d_available_cus; the rates are those of all 256).
#pragma once

namespace c2d_pr {
namespace {

// Tiles of rows x columns: 256 x 256, 128 x 256, 128 x 128, 64 x 64 with two groups of waves that share the contraction;
// from registers (products_few.h) 32 x 32, 16 x 16 by eight waves, 16 x 32 by two.
enum Shape { T256, T128W, T128, T64, T32, T16, T16W };

// Rounds in which `slots` resident workgroups make that many tiles.  A last one that is at most half full is made of halves
// (products_place.h), two workgroups a tile: 0.39 to 0.41 of a round where it is an eighth to a quarter full, 0.54 where it is
// half full (4500, 5000 and 6000 x 4096 in 256 x 256 tiles, contractions of 4096 in bf16 and in 8 bits).
inline double rounds_of(double tiles, double slots, bool halves) {
  if (tiles <= slots) return 1.0;
  const double whole = (double)(long long)(tiles / slots), rest = tiles / slots - whole;
  return whole + (rest < 0.02 ? 0.0 : halves && rest <= 0.5 ? 0.35 + 0.4 * rest : 1.0);
}

// Up to 16 rows a group.  Few column tiles: 16 columns a workgroup and its eight waves on one chain of segments each, to
// fill the chip and shorten the chains; many: 32 columns and two waves, whose starts and joins then weigh
// less (us, 8 waves of 16 columns / 2 waves of 32):  1 x 8192 x 4096 in 8 bits 8.1 / 9.4, 16 x 4096 x 4096 7.7 /
// 10.2;  64 rows in 64 groups, 2048 x 1024: in 8 bits 40.6 / 18.3, bf16 43.7 / 32.6.
inline Shape sixteen_rows_shape(int rows, int n, int groups, bool fp32, int cus) {
  const double tiles = (rows / 16.0 + 0.6 * groups) * ((n + 15) / 16);
  return !fp32 && tiles > 700.0 / 256 * cus ? T16W : T16;
}

// ---- grouped rows, bf16 and fp32
//
//   rows, bf16                    a round   a stage             measured (us)
//   256 x 256 tiles, from half of     6      1.12 .. 1.65        8192 x 8192 x 8192: 851, in 128 x 128 tiles 1045;
//     the CUs to all, and more                                   32 groups of 512 x 2048 x 2048: 173, 199
//     input gradient                  6      1.3 .. 1.65         8 groups of 625 x 1000 x 1536: 29.3, 128 x 128 30.6
//   128 x 256, in one round         3.5      0.7 .. 1.03         4500 rows of 4 groups, 1024 x 2048: 27.4, 128 x 128 29.9,
//                                                                256 x 256 41.9; 4096 x 4096 x 4096, two rounds: 128, 256 x 256 110
//     input gradient                3.5      0.85 .. 1.1         4292 rows of 3 groups, 1880 x 1512: 34.1, 128 x 128 38.2,
//                                                                256 x 256 48.1
//   128 x 128, one per CU           3.5      0.57                8 groups of 512 x 1024 x 1024: 17.4, 256 x 256 25.9,
//     up to two, and more           3.5      0.82 .. 1.04        64 x 64 31
//     input gradient                3.5      0.66                4096 x 2048 x 2048 in one group: 39.3, 256 x 256 48.8,
//       up to two, and more         3.5      0.87 .. 1.15        128 x 256 37.5
//   64 x 64, two K groups           3.0      0.25                 8 groups of 32 x 1024 x 1024: 7.0, 128 x 128 11.7
//   32 x 32 from registers          2.5      0.29                 (forward alone)
// Up to 16 rows a group, forward: 16 x 16 from registers.  fp32 is bound by its matrix instructions (a stage of a
// 64 x 64 tile 0.56, of 128 x 128 1.9 or, two per CU, 3.8) and has no 256 x 256 tiles, which gain 2.5 % on
// 4096^3 and lose wherever tiles are few (4 groups of 1024 x 416 x 1024: 241 against 42 in 64 x 64 tiles).
// (n, k: the result's columns and the contraction)
inline Shape rows_shape(int rows, int n, int k, int groups_, int es, bool forward, bool vec, int cus) {
  const int groups = groups_ < rows ? groups_ : rows;
  if (forward && (long long)rows <= 16ll * groups) return sixteen_rows_shape(rows, n, groups, es == 4, cus);
  // One group's row tiles are known.  Of several a last tile counts for what it costs, on average, and to a round of 128
  // rows a twentieth is added, since a few tiles too many cost another one (8 groups of 625 x 1000 x 1536, input
  // gradient, 258 tiles of 128 x 256: 33.5 us, in 256 x 256 tiles 29.3; of those more are made as halves).
  const double spare = groups == 1 ? 1.0 : 1.05;
  auto tiles = [&](int side, int columns) {
    const double down = groups == 1 ? (rows + side - 1) / side : (double)rows / side + 0.4 * groups;
    return down * ((n + columns - 1) / columns);
  };
  const double stages = ((long long)k * es + 127) / 128;
  const double t256 = tiles(256, 256), t128w = tiles(128, 256), t128 = tiles(128, 128);
  // From `lo` at half of `full` to `hi` at all of it, and behind.
  auto between = [](double t, double full, double lo, double hi) { return t >= full ? hi : t <= full / 2 ? lo : lo + (hi - lo) * (2 * t / full - 1); };
  const double us256 = rounds_of(t256, cus, true) * (between(t256, cus, forward ? 1.12 : 1.3, 1.65) * stages + 6.0);
  const double us128w = spare * t128w <= cus ? (forward ? between(t128w, cus, 0.7, 1.03) : between(t128w, cus, 0.85, 1.1)) * stages + 3.5 : 1e30;
  const double one = es == 4 ? 1.9 : forward ? 0.57 : 0.66;
  const double more = es == 4 ? between(t128, 2 * cus, 1.9, 3.8) : forward ? between(t128, 2 * cus, 0.82, 1.04) : between(t128, 2 * cus, 0.87, 1.15);
  const double us128 = rounds_of(spare * t128, 2 * cus, true) * ((t128 <= cus ? one : more) * stages + 3.5);
  const double us64 = rounds_of(tiles(64, 64), cus, false) * ((es == 4 ? 0.56 : 0.25) * stages + 3.0);
  const double us32 = forward ? tiles(32, 32) / cus * (es == 4 ? 0.4 : 0.29) * stages + 2.5 : 1e30;
  const double rest = us64 <= us32 ? us64 : us32, most = us128 <= rest ? us128 : rest;
  if (es == 2 && vec && us256 <= us128w && us256 <= most) return T256;
  if (es == 2 && vec && us128w <= most) return T128W;
  if (us128 <= us64 && us128 <= us32) return T128;
  return us64 <= us32 ? T64 : T32;
}

// ---- 8 bits
//
//                             a round   a block of k     measured, rows x n x k: this, and the next larger / smaller
//   256 x 256 tiles             3.5       1.95           8192 x 8192 x 8192: 509, in 128 x 128 tiles 680
//   128 x 128, two per CU       3.5       1.30  (0.75    1024 x 4096 x 4096:  27, in 256 x 256 tiles 53
//                                          one per CU)    2000 x 2000 x 256:  7.4, in 64 x 64 tiles 15.7
//   64 x 64, two K groups       3.5       0.28           256 x 4096 x 4096: 13.6, in 128 x 128 tiles 27.5
//                                                        2000 x 416 x 1024:  6.2, in 128 x 128 tiles 10.2
//   32 x 32 from registers      2.5       0.29           256 x 1024 x 1024:  4.9, in 64 x 64 tiles 6.0
// Up to 16 rows a group, 16-row tiles from registers: the weights' way is all there is (1 x 8192 x 4096: 8.1 us,
// 64 x 64 tiles 12.4; 16 x 4096 x 4096: 7.7 against 12.5).  An fp32 result doubles the matrix instructions and the
// registers of a block's products; it has no 256 x 256 tiles, whose registers it would spill, nor have
// operands that pass through registers on their way to LDS.
inline Shape fp8_shape(int rows, int n, int k, int groups_, bool ragged, bool out16, bool vec, int cus) {
  const int groups = !ragged ? 1 : groups_ < rows ? groups_ : rows;
  if ((long long)rows <= 16ll * groups) return sixteen_rows_shape(rows, n, groups, false, cus);
  auto tiles = [&](int side) {  // (a group's last row tile counts for what it costs, on average)
    const double down = ragged ? (double)rows / side + 0.4 * groups : (double)((rows + side - 1) / side);
    return down * ((n + side - 1) / side);
  };
  const double kb = (double)(((long long)k + 127) / 128), wide = out16 ? 1.0 : 1.5;
  const double t256 = tiles(256), t128 = tiles(128);
  const double us256 = rounds_of(t256, cus, true) * ((t256 <= cus ? 1.5 : 1.95) * kb + 3.5);
  const double us128 = rounds_of(t128, 2 * cus, true) * ((t128 <= cus ? 0.75 : 1.3) * wide * kb + 3.5);
  const double us64 = rounds_of(tiles(64), cus, false) * (0.28 * wide * kb + 3.5);
  const double us32 = tiles(32) / cus * 0.29 * kb + 2.5;
  if (out16 && vec && us256 <= us128 && us256 <= us64 && us256 <= us32) return T256;
  if (us128 <= us64 && us128 <= us32) return T128;
  return us64 <= us32 ? T64 : T32;
}

// ---- weight gradient
//
// The rows of a group are the contraction, dealt to `splits` workgroups where the tiles of dw are few; a round ends with
// the tile's way to memory, and splits with the sum over them.  The rounds are those of the whole chip: a plan that followed
// c2d_set_available_cus would change the workspace under a program that keeps one.
struct WgradPlan { int side, splits; };
inline WgradPlan wgrad_plan(int groups, int rows, int n, int k, int es) {
  const double stages = ((double)rows / groups * es + 127) / 128, mb = 4e-6 * groups * n * k;
  WgradPlan best = {64, 1};
  double least = 1e30;
  for (int side = es == 2 ? 256 : 128; side >= 64; side /= 2) {
    const double tiles = (double)groups * ((n + side - 1) / side) * ((k + side - 1) / side);
    const double slots = side == 128 ? 512 : 256;
    const double stage = es == 4 ? (side == 128 ? 3.8 : 0.56) : side == 256 ? 1.7 : side == 128 ? 1.2 : 0.27;
    const double round = side == 256 ? 20 : side == 128 ? 11 : 4;
    for (int splits = 1; splits == 1 || (splits <= 32 && 4 * splits <= stages && splits * mb <= 256); splits *= 2) {
      const double one = side == 128 && tiles * splits <= 256 ? 0.6 : 1.0;  // (one workgroup per CU)
      const double t = rounds_of(tiles * splits, slots, false) * one * (stage * stages / splits + round) +
                       (splits > 1 ? 4.0 + (splits + 1) * mb / 4.0 : 0.0);
      if (t < least) { least = t; best = {side, splits}; }
    }
  }
  return best;
}

}  // namespace
}  // namespace c2d_pr
