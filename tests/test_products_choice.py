"""Which kernel a product takes (csrc/products_choice.h, compiled for the host), and that the sizes which the GPU tests run reach
every kernel."""
import ctypes
import os
import subprocess

import pytest

from cap2det_amd import _lib
from tests import products_cases as cases

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")
SHAPES = ("256", "128w", "128", "64", "32", "16", "16w")

SOURCE = r"""
#include "products_choice.h"
using namespace c2d_pr;
extern "C" int fp8(int rows, int n, int k, int groups, int ragged, int out16, int vec, int cus) {
  return fp8_shape(rows, n, k, groups, ragged, out16, vec, cus);
}
extern "C" int rows_of(int rows, int n, int k, int groups, int es, int forward, int vec, int cus) {
  return rows_shape(rows, n, k, groups, es, forward, vec, cus);
}
extern "C" void wgrad(int groups, int rows, int n, int k, int es, int* side, int* splits) {
  const WgradPlan p = wgrad_plan(groups, rows, n, k, es);
  *side = p.side; *splits = p.splits;
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
  d = tmp_path_factory.mktemp("choice")
  (d / "choice.cpp").write_text(SOURCE)
  subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, "-o", str(d / "choice.so"), str(d / "choice.cpp")])
  return ctypes.CDLL(str(d / "choice.so"))


def _rows(counts):
  return cases.GAP + sum(counts) + cases.TAIL


def _wgrad(host, groups, rows, n, k, es):
  side, splits = ctypes.c_int(), ctypes.c_int()
  host.wgrad(groups, rows, n, k, es, ctypes.byref(side), ctypes.byref(splits))
  return side.value, splits.value


def test_the_8_bit_cases_reach_every_kernel(host):
  reached = set()
  for out16 in (0, 1):
    for vec in (0, 1):
      for m, n, k in cases.FP8_DENSE:
        reached.add((0, out16, vec, SHAPES[host.fp8(m, n, k, 1, 0, out16, vec, 256)]))
      for counts, n, k in cases.FP8_GROUPED:
        reached.add((1, out16, vec, SHAPES[host.fp8(_rows(counts), n, k, len(counts), 1, out16, vec, 256)]))
  every = {(ragged, out16, vec, shape) for ragged in (0, 1) for out16 in (0, 1) for vec in (0, 1)
           for shape in ("128", "64", "32", "16", "16w") + (("256",) if out16 and vec else ())}
  assert reached == every, every - reached


def test_the_grouped_cases_reach_every_kernel(host):
  reached = set()
  for forward in (0, 1):
    for es in (2, 4):
      for vec in (0, 1):
        for counts, n, k in cases.ROWS:
          reached.add((forward, es, vec, SHAPES[host.rows_of(_rows(counts), n, k, len(counts), es, forward, vec, 256)]))
  every = {(forward, es, vec, shape) for forward in (0, 1) for es in (2, 4) for vec in (0, 1)
           for shape in ("128", "64") + (("256", "128w") if es == 2 and vec else ()) + (("32", "16") if forward else ()) +
           (("16w",) if forward and es == 2 else ())}
  assert reached == every, every - reached


def test_the_weight_gradient_cases_reach_every_kernel(host):
  reached = set()
  for es in (2, 4):
    for counts, n, k in cases.WGRAD:
      side, splits = _wgrad(host, len(counts), _rows(counts), n, k, es)
      reached.add((es, side, splits > 1))
  every = {(es, side, split) for es in (2, 4) for side in ((256, 128, 64) if es == 2 else (128, 64)) for split in (False, True)}
  assert reached == every, every - reached


def test_the_plan_of_a_weight_gradient_is_the_workspace(host):
  lib = _lib.load()
  for kind, es in ((0, 4), (1, 2)):
    for counts, n, k in cases.WGRAD:
      rows, groups = _rows(counts), len(counts)
      splits = _wgrad(host, groups, rows, n, k, es)[1]
      assert lib.c2dp_grouped_matmul_wgrad_workspace_bytes(groups, rows, n, k, kind) == (4 * splits * groups * n * k if splits > 1 else 0)


def test_fewer_cus_are_fewer_workgroups_a_round(host):
  """Half the tiles on half the CUs are the same rounds: the same kernel (c2d_set_available_cus; the placement counts by it
  too)."""
  sizes = [(rows, n, k) for rows in (8, 64, 256, 512, 1024, 2304, 4096, 5120) for n in (64, 416, 1000, 2048, 4096) for k in (128, 512, 2048)]
  differs = 0
  for rows, n, k in sizes:
    for cus in (128, 64):
      part = 256 // cus
      for vec in (0, 1):
        for out16 in (0, 1):
          a = host.fp8(rows, n, k, 1, 0, out16, vec, cus)
          assert rows <= 16 or rows % 256 or a == host.fp8(rows * part, n, k, 1, 0, out16, vec, 256)
          differs += a != host.fp8(rows, n, k, 1, 0, out16, vec, 256)
        for es in (2, 4):
          for forward in (0, 1):
            a = host.rows_of(rows, n, k, 1, es, forward, vec, cus)
            assert rows <= 16 or rows % 256 or a == host.rows_of(rows * part, n, k, 1, es, forward, vec, 256)
            differs += a != host.rows_of(rows, n, k, 1, es, forward, vec, 256)
  assert differs > 100
