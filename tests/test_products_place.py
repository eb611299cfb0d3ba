"""Where the workgroups of a grouped product lie (csrc/products_place.h), compiled for the host: every row and column tile
is made once, halves of tiles are halves, and what has no tile clears the rows of no group."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

from cap2det_amd import _lib
from tests import util_products as up

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")

# place_tile of products_common.h with the wave's scans as loops
SOURCE = r"""
#include "products_place.h"
using namespace c2d_pr;
template <int BM, bool H>
static void place(const int* lo, const int* hi, int groups, bool ragged, int rows, int ntiles, unsigned bid, unsigned nbid,
                  int slots, int* out) {
  Place p = {};
  int full = 0, half = 0;
  if (!ragged) full = (rows + BM - 1) / BM;
  else for (int e = 0; e < groups; ++e) { full += full_tiles_of<BM, H>(hi[e] - lo[e]); half += half_tiles_of<BM, H>(hi[e] - lo[e]); }
  const Pick t = pick_tile<H>(p, full, half, ntiles, bid, nbid, slots);
  if (p.live && !ragged) {
    p.lo = 0; p.hi = rows;
    tile_rows<BM>(p, t, 0, full);
  } else if (p.live) {
    int before = 0;
    for (int e = 0; e < groups; ++e) {
      const int fulls = full_tiles_of<BM, H>(hi[e] - lo[e]), mine = t.small ? half_tiles_of<BM, H>(hi[e] - lo[e]) : fulls;
      if (before + mine > t.mt) {
        p.e = e; p.lo = lo[e]; p.hi = hi[e];
        tile_rows<BM>(p, t, before, fulls);
        break;
      }
      before += mine;
    }
  }
  const int v[9] = {p.live, p.e, p.m0, p.hi, p.nt, t.halved, t.small, p.spare, p.spares};
  for (int i = 0; i < 9; ++i) out[i] = v[i];
}
extern "C" unsigned place_all(int bm, int halves, const int* lo, const int* hi, int groups, int ragged, int rows, int ntiles,
                              int slots, int* out, unsigned room) {
  const unsigned n = place_grid(bm, groups, ragged, rows, ntiles, halves ? slots / 2 : 0);
  if (n > room) return 0;
  for (unsigned b = 0; b < n; ++b) {
    int* o = out + 9 * b;
#define AT(BM, H) if (bm == BM && (halves != 0) == H) place<BM, H>(lo, hi, groups, ragged, rows, ntiles, b, n, slots, o)
    AT(16, false); AT(32, false); AT(64, false); AT(128, false); AT(128, true); AT(256, true);
  }
  return n;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
  d = tmp_path_factory.mktemp("place")
  (d / "place.cpp").write_text(SOURCE)
  subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, "-o", str(d / "place.so"), str(d / "place.cpp")])
  return ctypes.CDLL(str(d / "place.so"))


def _place(host, bm, halves, offsets, rows, n, bn, slots):
  ntiles = -(-n // bn)
  ragged = offsets is not None
  spans = np.array(up.spans(offsets, rows) if ragged else [(0, rows)], np.int32)
  lo, hi = np.ascontiguousarray(spans[:, 0]), np.ascontiguousarray(spans[:, 1])
  ptr = lambda a: a.ctypes.data_as(ctypes.POINTER(ctypes.c_int))
  out = np.zeros((1 << 17, 9), np.int32)
  count = host.place_all(bm, int(halves), ptr(lo), ptr(hi), len(spans), int(ragged), rows, ntiles, slots, ptr(out), len(out))
  assert count and count % 8 == 0
  return spans, ntiles, out[:count]


def _check(host, bm, halves, offsets, rows, n, bn, slots):
  """Returns how many workgroups made a half of a full tile."""
  spans, ntiles, out = _place(host, bm, halves, offsets, rows, n, bn, slots)
  made = np.zeros((rows, ntiles), np.int32)
  for live, e, m0, hi, nt, halved, small, spare, spares in out:
    if not live:
      continue
    height = bm // 2 if halves and hi - m0 <= bm // 2 else bm             # (the kernels' rule)
    assert not (halved or small) or height == bm // 2, (e, m0, hi)
    lo_e, hi_e = spans[e]
    assert lo_e <= m0 < hi <= hi_e and 0 <= nt < ntiles
    made[m0:min(hi, m0 + height), nt] += 1
  inside = np.zeros(rows, bool)
  for lo, hi in spans:
    inside[lo:hi] = True
  assert (made[inside] == 1).all() and (made[~inside] == 0).all()
  spare = np.sort(out[(out[:, 0] == 0) & (out[:, 7] >= 0), 7])
  if offsets is not None:
    assert out[0, 8] > 0 and np.array_equal(spare, np.arange(out[0, 8]))
  return int(((out[:, 0] != 0) & (out[:, 5] != 0)).sum())


# tile height, halves, tile width, resident workgroups of an XCD
SHAPES = [(256, True, 256, 32), (128, True, 256, 32), (128, True, 128, 64), (64, False, 64, 32), (32, False, 32, 1), (16, False, 16, 1),
          (256, True, 256, 28), (128, True, 128, 1)]


@pytest.mark.parametrize("bm,halves,bn,slots", SHAPES)
def test_one_group_and_no_groups(host, bm, halves, bn, slots):
  for rows in (1, bm // 2, bm // 2 + 1, bm, bm + 1, 3 * bm - 1, 4500):
    for n in (1, bn, 5 * bn + 1):
      _check(host, bm, halves, None, rows, n, bn, slots)
      _check(host, bm, halves, [0, rows], rows, n, bn, slots)


@pytest.mark.parametrize("rows,n", [(4500, 4096), (8400, 2048), (9000, 4096), (4096 + 300, 4096)])
@pytest.mark.parametrize("ragged", [False, True])
def test_the_last_round_of_one_long_group_is_made_as_halves(host, rows, n, ragged):
  assert _check(host, 256, True, [0, rows] if ragged else None, rows, n, 256, 32) > 0


@pytest.mark.parametrize("bm,halves,bn,slots", SHAPES)
def test_ragged_groups(host, bm, halves, bn, slots):
  r = random.Random(bm + bn + slots)
  cut = 0
  for _ in range(40):
    groups = r.choice((1, 2, 5, 32, 70, 150))
    rows = r.randrange(1, 9000)
    cuts = sorted(r.randrange(0, rows + 1) for _ in range(groups + 1))
    for offsets in (cuts, [0] + cuts[1:-1] + [rows], r.sample(cuts, len(cuts)), [o * 3 - rows for o in cuts]):
      cut += _check(host, bm, halves, offsets, rows, r.choice((64, 1000, 2048)), bn, slots)
  assert cut > 0 or not halves or slots == 1
