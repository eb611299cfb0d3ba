// Where a workgroup's tile lies among the groups of rows: plain arithmetic, the same on the host and on the device.
#pragma once
#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define C2D_PR_HD __host__ __device__ __forceinline__
#else
#define C2D_PR_HD inline
#endif

namespace c2d_pr {
namespace {

C2D_PR_HD int lesser(int a, int b) { return a < b ? a : b; }
C2D_PR_HD int larger(int a, int b) { return a < b ? b : a; }

// Group boundaries as they are used: each offset clamped to [0, rows], and at least every earlier one.
struct Span { int lo, hi; };

struct Place {
  int e, lo, hi;   // the tile's group and its rows (a half of a tile: hi is that half's end)
  int m0, nt;      // first row of the tile, column tile
  bool live;       // false: the workgroup has no tile
  int begin, end;  // rows outside [begin, end) are in no group
  int spare, spares;  // a workgroup without a tile: its number among those that clear rows (-1: none)
};

// Row tiles of BM rows that a group of r rows makes.  HALVES: a last one of BM / 2 rows or less is counted apart.
template <int BM, bool HALVES>
C2D_PR_HD int full_tiles_of(int r) { return HALVES ? (r + BM / 2 - 1) / BM : (r + BM - 1) / BM; }
template <int BM, bool HALVES>
C2D_PR_HD int half_tiles_of(int r) { return (r + BM - 1) / BM - full_tiles_of<BM, HALVES>(r); }

// A tile by its number: row tile `mt` of all groups' full ones, or (small) of all groups' halves; halved: the first or
// the second half of a full one.
struct Pick {
  int mt;
  bool small, halved, second;
};

// Tile of workgroup `bid` out of `nbid` (a multiple of 8), of `full` and `half` row tiles by `ntiles` column tiles.
// Workgroups go round the 8 XCDs by number; XCD x takes the x-th eighth of the tiles, in bands of 4 row tiles by all
// column tiles, so that what runs there at a time shares rows and weights in that XCD's L2.
// HALVES: a tile of BM / 2 rows or less costs half, and a group's last one often is.  All of those come behind the
// others; and where the others end with a round that would leave most of an XCD's `slots` resident
// workgroups without a tile, the tiles of that round are made as halves too, by two workgroups each.
// Sets p.nt, p.live, p.spare and p.spares.
template <bool HALVES>
C2D_PR_HD Pick pick_tile(Place& p, int full, int half, int ntiles, unsigned bid, unsigned nbid, int slots) {
  Pick t = {0, false, false, false};
  const int xcd = bid & 7, local = bid >> 3, per = nbid >> 3;
  const int full_tiles = full * ntiles, half_tiles = half * ntiles;
  const int my_full = (full_tiles + 7 - xcd) >> 3, my_half = (half_tiles + xcd) >> 3;
  const int over = my_full % slots;
  const int cut = HALVES && my_full > slots && 2 * over + my_half <= slots ? over : 0;
  p.live = local < my_full + cut + my_half;
  p.spares = 8 * (per - ((full_tiles + 7) >> 3) - ((half_tiles + 7) >> 3) - (HALVES ? slots / 2 : 0));
  p.spare = -1;
  if (!p.live) {
    const int spare = 8 * (local - my_full - cut - my_half) + xcd;
    if (spare < p.spares) p.spare = spare;
    return t;
  }
  // the tile among those of its kind: whole eighths before this XCD's, of which the first (last) few have one more
  t.small = HALVES && local >= my_full + cut;
  t.halved = local >= my_full - cut && !t.small && cut > 0;
  const int nth = t.small ? local - my_full - cut : t.halved ? my_full - cut + ((local - my_full + cut) >> 1) : local;
  t.second = t.halved && ((local - my_full + cut) & 1);
  const int idx = t.small ? xcd * (half_tiles >> 3) + larger(0, xcd - 8 + (half_tiles & 7)) + nth
                          : xcd * (full_tiles >> 3) + lesser(xcd, full_tiles & 7) + nth;
  constexpr int BAND = 4;
  const int mtiles = t.small ? half : full;
  const int band = idx / (BAND * ntiles), at = idx - band * BAND * ntiles;
  const int bm = lesser(BAND, mtiles - band * BAND);
  t.mt = band * BAND + at % bm;
  p.nt = at / bm;
  return t;
}

// Rows of the picked tile in its group [p.lo, p.hi), `before` full tiles lying in front of the group's.  Half of a tile
// ends where the tile's other half begins or where the tile ends, not where the group does.
template <int BM>
C2D_PR_HD void tile_rows(Place& p, const Pick& t, int before, int full_of_group) {
  p.m0 = p.lo + (t.small ? full_of_group : t.mt - before) * BM;
  if (t.halved) {
    if (t.second) p.m0 += BM / 2;
    p.hi = lesser(p.hi, p.m0 + BM / 2);
    p.live = p.m0 < p.hi;
  }
}

// The largest number of workgroups that placing can need, with some to spare that clear rows; 0: too many.
// `cut`: tiles of an XCD that may be made as halves.
inline unsigned place_grid(int BM, int groups, bool ragged, int rows, int ntiles, int cut) {
  const long long mt = ragged ? (long long)rows / BM + (groups < rows ? groups : rows) : ((long long)rows + BM - 1) / BM;
  const long long n = ((mt * ntiles + 7) / 8 + cut + (ragged ? 8 : 0)) * 8;
  return n < (1ll << 30) ? (unsigned)n : 0u;
}

}  // namespace
}  // namespace c2d_pr
