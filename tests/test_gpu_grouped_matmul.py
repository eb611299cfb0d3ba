"""Matrix products grouped by expert against 64-bit oracles: forward, input gradient, weight gradient."""
import pytest
import torch

from cap2det_amd import hip_ops as ops
from tests import util_products as up

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN = float("nan")


def _gen(seed=0):
  return torch.Generator(device="cuda").manual_seed(seed)


def _offs(offsets):
  return torch.tensor(offsets, dtype=torch.int32, device="cuda")


def _same(got, want, rows=None):
  """Bit for bit what the exact sums round to; `rows`: the spans that count."""
  want = want.to(got.dtype)
  for lo, hi in (rows or [(0, got.shape[0])]):
    assert torch.equal(got[lo:hi], want[lo:hi]), (lo, hi, (got[lo:hi] != want[lo:hi]).nonzero()[:4].tolist())


# counts of the groups: none, one, a tile less one / exactly / and one more, long, in one and in many groups
COUNTS = [[1], [0], [0, 0, 5, 0], [127, 128, 129], [1] * 70, [300, 0, 1, 17], [2, 0, 0, 0, 0, 0, 0, 31, 64]]
# (n, k): below, at and above the tiles and stages; odd ones take element loads
SIZES = [(1, 1), (8, 8), (64, 64), (33, 40), (130, 264), (128, 128), (257, 72), (40, 1000), (7, 131), (300, 63)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "x".join(map(str, c[:9])))
def test_products_of_integers_are_exact(dtype, n, k, counts):
  """Sums of whole numbers below 2^24: every product, and no other, is in the result once."""
  gen = _gen(n * 1000 + k)
  tail = 3
  offsets = up.offsets_of(counts, first=2)
  t = offsets[-1] + tail
  x = up.integers(gen, (t, k), 8, dtype)
  dy = up.integers(gen, (t, n), 8, dtype)
  w = up.integers(gen, (len(counts), n, k), 8, dtype)
  offs, rows = _offs(offsets), up.spans(offsets, t)
  for got, want in ((ops.grouped_matmul(x, w, offs), up.grouped(x, w, offsets)),
                    (ops.grouped_matmul_dgrad(dy, w, offs), up.grouped(dy, w.transpose(1, 2), offsets))):
    assert got.dtype == dtype
    _same(got, want, rows)
    assert (got[:2] == 0).all() and (got[offsets[-1]:] == 0).all()
  dw = ops.grouped_matmul_wgrad(x, dy, offs)
  assert dw.dtype == F32
  _same(dw, up.grouped_dw(x, dy, offsets))
  if dtype == BF16:
    _same(ops.grouped_matmul(x, w, offs, out_dtype=F32), up.grouped(x, w, offsets), rows)
    _same(ops.grouped_matmul_dgrad(dy, w, offs, out_dtype=F32), up.grouped(dy, w.transpose(1, 2), offsets), rows)


@pytest.mark.parametrize("counts,n,k", [([700, 0, 1300], 520, 1032), ([4096], 256, 512), ([3] * 64, 384, 2048),
                                        ([16, 40, 0, 9], 1024, 4096), ([2000, 2000], 416, 1024),
                                        ([5000, 1, 3000], 1040, 1048)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_larger_products_of_integers_are_exact(dtype, counts, n, k):
  gen = _gen(7)
  offsets = up.offsets_of(counts)
  x = up.integers(gen, (offsets[-1], k), 4, dtype)
  dy = up.integers(gen, (offsets[-1], n), 4, dtype)
  w = up.integers(gen, (len(counts), n, k), 4, dtype)
  offs = _offs(offsets)
  _same(ops.grouped_matmul(x, w, offs), up.grouped(x, w, offsets))
  _same(ops.grouped_matmul_dgrad(dy, w, offs), up.grouped(dy, w.transpose(1, 2), offsets))
  _same(ops.grouped_matmul_wgrad(x, dy, offs), up.grouped_dw(x, dy, offsets))


# Sizes at which the estimated times choose 256 x 256 and (last) 128 x 256 tiles, with groups whose last tile is short, long and whole, more
# row tiles than an XCD holds at a time, and (5800 rows of 2048 columns) a last round that is made as halves
@pytest.mark.parametrize("counts,n,k", [([3000, 100, 5900], 2048, 1024), ([5800], 2048, 1024), ([600, 0, 130, 256, 2000, 385] * 2, 1100, 1032),
                                        ([37 * i % 299 for i in range(150)], 520, 1032), ([128] * 65 + [0, 1, 500], 1032, 264),
                                        ([1500, 1000, 1, 1999], 1024, 2048), ([1700, 0, 2592], 1880, 1512), ([4096], 2048, 2048)])
def test_large_tiles_of_integers_are_exact(counts, n, k):
  gen = _gen(21)
  offsets = up.offsets_of(counts, first=5)
  t = offsets[-1] + 40
  x, dy = up.integers(gen, (t, k), 4, BF16), up.integers(gen, (t, n), 4, BF16)
  w = up.integers(gen, (len(counts), n, k), 4, BF16)
  offs, rows = _offs(offsets), up.spans(offsets, t)
  for got, want in ((ops.grouped_matmul(x, w, offs), up.grouped(x, w, offsets)),
                    (ops.grouped_matmul(x, w, offs, out_dtype=F32), up.grouped(x, w, offsets)),
                    (ops.grouped_matmul_dgrad(dy, w, offs), up.grouped(dy, w.transpose(1, 2), offsets))):
    _same(got, want, rows)
    assert (got[:5] == 0).all() and (got[offsets[-1]:] == 0).all()
  _same(ops.grouped_matmul_wgrad(x, dy, offs), up.grouped_dw(x, dy, offsets))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("counts,n,k", [([8192], 512, 512), ([4000, 0, 1], 136, 264), ([3001], 65, 131), ([1000, 1, 2000, 700], 2048, 2048)])
def test_wgrad_of_long_groups_and_few_tiles(dtype, counts, n, k):
  """The rows of a group dealt to several workgroups (and, last, 256 x 256 tiles): exact, and added to what is there."""
  gen = _gen(22)
  offsets = up.offsets_of(counts)
  x, dy = up.integers(gen, (offsets[-1], k), 4, dtype), up.integers(gen, (offsets[-1], n), 4, dtype)
  want = up.grouped_dw(x, dy, offsets)
  _same(ops.grouped_matmul_wgrad(x, dy, _offs(offsets)), want)
  start = up.integers(gen, want.shape, 50)
  out = start.clone()
  ops.grouped_matmul_wgrad(x, dy, _offs(offsets), out=out, accumulate=True)
  _same(out, want + start.double())


def test_two_graphs_and_two_streams_share_no_workspace():
  """Weight gradients that take a workspace, captured twice and replayed beside each other and beside eager calls."""
  gen = _gen(23)
  offs = _offs([0, 8192])
  sets = []
  for _ in range(2):
    x = torch.randn(8192, 256, generator=gen, device="cuda").to(BF16)
    dy = torch.randn(8192, 192, generator=gen, device="cuda").to(BF16)
    out = torch.empty(1, 192, 256, device="cuda")
    want = ops.grouped_matmul_wgrad(x, dy, offs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      ops.grouped_matmul_wgrad(x, dy, offs, out=out)
    sets.append((x, dy, out, want, graph, torch.cuda.Stream()))
  for _ in range(5):
    torch.cuda.synchronize()
    eager = []
    for x, dy, out, want, graph, stream in sets:
      out.fill_(NAN)
      stream.wait_stream(torch.cuda.current_stream())
      with torch.cuda.stream(stream):
        graph.replay()
        eager.append(ops.grouped_matmul_wgrad(x, dy, offs))
    torch.cuda.synchronize()
    for (x, dy, out, want, graph, stream), again in zip(sets, eager):
      assert torch.equal(out, want) and torch.equal(again, want)


def test_a_step_plan_replays_the_products_on_other_tensors():
  from cap2det_amd.step_plan import StepPlan
  gen = _gen(24)
  offs = _offs([0, 30, 30, 100])
  x, dy = torch.randn(100, 72, generator=gen, device="cuda").to(BF16), torch.randn(100, 40, generator=gen, device="cuda").to(BF16)
  w = torch.randn(3, 40, 72, generator=gen, device="cuda").to(BF16)
  y, dx, dw = torch.empty(100, 40, device="cuda", dtype=BF16), torch.empty(100, 72, device="cuda", dtype=BF16), torch.empty(3, 40, 72, device="cuda")
  plan = StepPlan()
  plan.bind_tensor("x", x)
  plan.bind_tensor("dy", dy)
  with plan.recording():
    _layer(x, dy, w, offs, y, dx, dw)
  assert plan.calls == 3
  for _ in range(3):
    x2, dy2 = torch.randn_like(x), torch.randn_like(dy)
    for t in (y, dx, dw):
      t.fill_(NAN)
    plan.replay(dict(x=x2, dy=dy2), {})
    torch.cuda.synchronize()
    for got, want in zip((y, dx, dw), (ops.grouped_matmul(x2, w, offs), ops.grouped_matmul_dgrad(dy2, w, offs),
                                       ops.grouped_matmul_wgrad(x2, dy2, offs))):
      assert torch.equal(got, want)


def test_a_step_plan_keeps_its_workspaces_and_results():
  """Replays write into memory that nobody else has been given since the recording."""
  from cap2det_amd.step_plan import StepPlan
  gen = _gen(26)
  offs = _offs([0, 8192])
  x, dy = torch.randn(8192, 256, generator=gen, device="cuda").to(BF16), torch.randn(8192, 192, generator=gen, device="cuda").to(BF16)
  out, w = torch.empty(1, 192, 256, device="cuda"), torch.randn(1, 192, 256, generator=gen, device="cuda").to(BF16)
  want, y = ops.grouped_matmul_wgrad(x, dy, offs), ops.grouped_matmul(x, w, offs)
  plan = StepPlan()
  with plan.recording():
    ops.grouped_matmul_wgrad(x, dy, offs, out=out)
    ops.grouped_matmul(x, w, offs)
    ops.fp8_quantize(x)
  torch.cuda.synchronize()
  others = [torch.full((1 << e,), 7, dtype=torch.uint8, device="cuda") for e in range(12, 25) for _ in range(4)]
  for _ in range(3):
    out.fill_(NAN)
    plan.replay({}, {})
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(bool((t == 7).all()) for t in others)
  assert any(t.shape == y.shape and torch.equal(t, y) for t in plan.keep)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("counts,n,k", [([100, 0, 37], 200, 328), ([9, 3, 1, 0], 96, 640)])
def test_real_values_within_the_rounding_of_sums(dtype, counts, n, k):
  gen = _gen(3)
  offsets = up.offsets_of(counts)
  t = offsets[-1]
  x = torch.randn(t, k, generator=gen, device="cuda").to(dtype)
  dy = torch.randn(t, n, generator=gen, device="cuda").to(dtype)
  w = (torch.randn(len(counts), n, k, generator=gen, device="cuda") * k ** -0.5).to(dtype)
  offs = _offs(offsets)
  wt = w.transpose(1, 2)
  step = up.half_step(dtype)
  for got, want, mag, terms in (
      (ops.grouped_matmul(x, w, offs), up.grouped(x, w, offsets), up.grouped(x.abs(), w.abs(), offsets), k),
      (ops.grouped_matmul_dgrad(dy, w, offs), up.grouped(dy, wt, offsets), up.grouped(dy.abs(), wt.abs(), offsets), n)):
    up.assert_within(got, want, up.sum_bound(terms, mag) + step * want.abs() * (1 + 2.0 ** -20))
  mag = up.grouped_dw(x.abs(), dy.abs(), offsets)
  up.assert_within(ops.grouped_matmul_wgrad(x, dy, offs), up.grouped_dw(x, dy, offsets), up.sum_bound(max(counts), mag))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_against_differences(dtype):
  """The products are linear in each operand: <dx, e> and <dw, e> equal the differences of <y, dy> along e, exactly
  for whole numbers."""
  gen = _gen(11)
  offsets = up.offsets_of([5, 0, 12, 3])
  t, n, k = 20, 24, 40
  x, ex = (up.integers(gen, (t, k), 4, dtype) for _ in range(2))
  w, ew = (up.integers(gen, (4, n, k), 4, dtype) for _ in range(2))
  dy = up.integers(gen, (t, n), 4, dtype)
  offs = _offs(offsets)
  f = lambda x_, w_: (ops.grouped_matmul(x_, w_, offs, out_dtype=F32).double() * dy.double()).sum().item()
  dx = ops.grouped_matmul_dgrad(dy, w, offs, out_dtype=F32).double()
  dw = ops.grouped_matmul_wgrad(x, dy, offs).double()
  assert f(x + ex, w) - f(x, w) == (dx * ex.double()).sum().item()
  assert f(x, w + ew) - f(x, w) == (dw * ew.double()).sum().item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pitch,column", [(8, 0), (16, 8), (5, 1), (3, 0)])
def test_row_pitches_and_what_lies_beside_the_columns(dtype, pitch, column):
  """Views of wider matrices that hold NaN beside the operands' columns and marks beside the results'."""
  gen = _gen(5)
  offsets = up.offsets_of([37, 0, 130])
  t, n, k = 167, 72, 200
  x = up.integers(gen, (t, k), 8, dtype)
  dy = up.integers(gen, (t, n), 8, dtype)
  w = up.integers(gen, (3, n, k), 8, dtype)
  offs = _offs(offsets)
  xv = up.view_with_pitch(x, k + pitch, NAN, column)
  dyv = up.view_with_pitch(dy, n + pitch, NAN, column)
  for cols, want, f in ((n, up.grouped(x, w, offsets), lambda o: ops.grouped_matmul(xv, w, offs, out=o)),
                        (k, up.grouped(dy, w.transpose(1, 2), offsets), lambda o: ops.grouped_matmul_dgrad(dyv, w, offs, out=o))):
    big = torch.full((t, cols + pitch), 77.0, device="cuda").to(dtype)
    got = f(big[:, column:column + cols])
    _same(got, want)
    big[:, column:column + cols] = 77.0
    assert (big == 77.0).all()
  _same(ops.grouped_matmul_wgrad(xv, dyv, offs), up.grouped_dw(x, dy, offsets))


def test_rows_of_no_group_are_not_read_and_left_as_they_were():
  gen = _gen(6)
  offsets = [4, 9, 9, 30]
  t, n, k = 50, 40, 64
  for dtype in (BF16, F32):
    x = up.integers(gen, (t, k), 8, dtype)
    dy = up.integers(gen, (t, n), 8, dtype)
    x[:4], x[30:], dy[:4], dy[30:] = NAN, float("inf"), NAN, float("-inf")
    w = up.integers(gen, (3, n, k), 8, dtype)
    offs, rows = _offs(offsets), up.spans(offsets, t)
    out = torch.full((t, n), 5.0, device="cuda").to(dtype)
    _same(ops.grouped_matmul(x, w, offs, out=out), up.grouped(x, w, offsets), rows)
    assert (out[:4] == 5.0).all() and (out[30:] == 5.0).all()
    out = torch.full((t, k), 5.0, device="cuda").to(dtype)
    _same(ops.grouped_matmul_dgrad(dy, w, offs, out=out), up.grouped(dy, w.transpose(1, 2), offsets), rows)
    assert (out[:4] == 5.0).all() and (out[30:] == 5.0).all()
    dw = ops.grouped_matmul_wgrad(x, dy, offs)
    _same(dw, up.grouped_dw(x, dy, offsets))
    # the rows of no group in a fresh result
    y = ops.grouped_matmul(x, w, offs)
    assert (y[:4] == 0).all() and (y[30:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(72, 136), (41, 67)])
def test_nan_and_infinity_stay_in_their_rows_and_groups(dtype, n, k):
  gen = _gen(8)
  offsets = up.offsets_of([33, 20, 40])
  t = 93
  x = up.integers(gen, (t, k), 8, dtype)
  dy = up.integers(gen, (t, n), 8, dtype)
  w = up.integers(gen, (3, n, k), 8, dtype)
  offs = _offs(offsets)
  bad = x.clone()
  bad[32], bad[60, 3] = NAN, float("inf")
  y = ops.grouped_matmul(bad, w, offs)
  want = up.grouped(x, w, offsets)
  dy[60] = dy[60] + (dy[60] == 0)
  keep = torch.ones(t, dtype=torch.bool, device="cuda")
  keep[32] = keep[60] = False
  _same(y[keep], want[keep])
  assert y[32].isnan().all() and not y[60].isfinite().any()
  # a group's weights reach that group's rows alone, a row the gradient of its group alone
  wbad = w.clone()
  wbad[1] = NAN
  y = ops.grouped_matmul(x, wbad, offs)
  _same(torch.cat([y[:33], y[53:]]), torch.cat([want[:33], want[53:]]))
  assert y[33:53].isnan().all()
  dw, dw_want = ops.grouped_matmul_wgrad(bad, dy, offs), up.grouped_dw(x, dy, offsets)
  _same(dw[1], dw_want[1])
  assert dw[0].isnan().all()
  others = [j for j in range(k) if j != 3]     # (row 60, the infinity in column 3, is the third group's)
  _same(dw[2][:, others], dw_want[2][:, others])
  assert not dw[2][:, 3].isfinite().any()


@pytest.mark.parametrize("offsets", [[-5, 10, 200], [0, 30, 10, 25, 64], [64, 0, 64], [7, 7, 7], [-2 ** 31, 2 ** 31 - 1], [10, 5, 2]])
def test_offsets_that_do_not_rise_or_reach_outside(offsets):
  """Clamped to [0, rows] and to the largest before them: groups stay disjoint and inside."""
  gen = _gen(9)
  t, n, k = 64, 40, 72
  groups = len(offsets) - 1
  x = up.integers(gen, (t, k), 8, BF16)
  dy = up.integers(gen, (t, n), 8, BF16)
  w = up.integers(gen, (groups, n, k), 8, BF16)
  offs, rows = _offs(offsets), up.spans(offsets, t)
  for got, want in ((ops.grouped_matmul(x, w, offs), up.grouped(x, w, offsets)),
                    (ops.grouped_matmul_dgrad(dy, w, offs), up.grouped(dy, w.transpose(1, 2), offsets))):
    _same(got, want, rows)
    assert (got[want.isnan().any(1)] == 0).all()
  _same(ops.grouped_matmul_wgrad(x, dy, offs), up.grouped_dw(x, dy, offsets))


@pytest.mark.parametrize("t,n,k", [(0, 16, 24), (5, 0, 24), (5, 16, 0), (0, 0, 0)])
def test_empty_sizes(t, n, k):
  for dtype in (BF16, F32):
    x, dy = torch.ones(t, k, device="cuda", dtype=dtype), torch.ones(t, n, device="cuda", dtype=dtype)
    w = torch.ones(2, n, k, device="cuda", dtype=dtype)
    offs = _offs([0, t // 2, t])
    assert torch.equal(ops.grouped_matmul(x, w, offs), torch.full((t, n), float(k), device="cuda").to(dtype))
    assert torch.equal(ops.grouped_matmul_dgrad(dy, w, offs), torch.full((t, k), float(n), device="cuda").to(dtype))
    dw = ops.grouped_matmul_wgrad(x, dy, offs)
    assert dw.shape == (2, n, k) and (t > 0 or (dw == 0).all())


@pytest.mark.parametrize("n,k", [(72, 136), (41, 67)])
def test_wgrad_accumulates(n, k):
  gen = _gen(10)
  offsets = up.offsets_of([33, 0, 140])
  x, dy = up.integers(gen, (173, k), 8, BF16), up.integers(gen, (173, n), 8, BF16)
  start = up.integers(gen, (3, n, k), 50)
  out = start.clone()
  got = ops.grouped_matmul_wgrad(x, dy, _offs(offsets), out=out, accumulate=True)
  assert got is out
  _same(out, up.grouped_dw(x, dy, offsets) + start.double())
  ops.grouped_matmul_wgrad(x, dy, _offs(offsets), out=out)
  _same(out, up.grouped_dw(x, dy, offsets))


def _layer(x, dy, w, offs, y, dx, dw):
  ops.grouped_matmul(x, w, offs, out=y)
  ops.grouped_matmul_dgrad(dy, w, offs, out=dx)
  ops.grouped_matmul_wgrad(x, dy, offs, out=dw)


def test_the_same_bits_every_time_on_another_stream_and_in_a_replayed_graph():
  gen = _gen(12)
  offsets = up.offsets_of([600, 0, 37, 900])
  t, n, k = 1537, 200, 264
  x = torch.randn(t, k, generator=gen, device="cuda").to(BF16)
  dy = torch.randn(t, n, generator=gen, device="cuda").to(BF16)
  w = torch.randn(4, n, k, generator=gen, device="cuda").to(BF16)
  offs = _offs(offsets)
  want = (ops.grouped_matmul(x, w, offs), ops.grouped_matmul_dgrad(dy, w, offs), ops.grouped_matmul_wgrad(x, dy, offs))
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    again = (ops.grouped_matmul(x, w, offs), ops.grouped_matmul_dgrad(dy, w, offs), ops.grouped_matmul_wgrad(x, dy, offs))
  torch.cuda.current_stream().wait_stream(side)
  for a, b in zip(want, again):
    assert torch.equal(a, b)
  outs = [torch.empty_like(v) for v in want]
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    _layer(x, dy, w, offs, *outs)
  for i in range(4):
    # other inputs, other group lengths, eager work between the replays
    x.copy_(torch.randn(t, k, generator=gen, device="cuda"))
    dy.copy_(torch.randn(t, n, generator=gen, device="cuda"))
    offs.copy_(_offs(up.offsets_of([100 * i, 500, 0, 1537 - 500 - 100 * i])))
    for o in outs:
      o.fill_(NAN)
    graph.replay()
    torch.cuda.synchronize()
    eager = (ops.grouped_matmul(x, w, offs), ops.grouped_matmul_dgrad(dy, w, offs), ops.grouped_matmul_wgrad(x, dy, offs))
    for a, b in zip(outs, eager):
      assert torch.equal(a, b)


def test_rows_behind_two_gigabytes_and_four():
  """x is 4.4 GB: row offsets that pass 32 bits, in the forward product and along the weight gradient's sum."""
  t, n, k = 1100000, 8, 2000
  offsets = [0, 5, 536000, 1099990]
  gen = _gen(13)
  x = torch.zeros(t, k, device="cuda", dtype=BF16)
  at = [0, 4, 5, 300000, 535999, 536000, 536900, 1073800, 1099989, 1099995]
  x[at] = up.integers(gen, (len(at), k), 8, BF16)
  dy = up.integers(gen, (t, n), 8, BF16)
  w = up.integers(gen, (3, n, k), 8, BF16)
  offs = _offs(offsets)
  y = ops.grouped_matmul(x, w, offs)
  want = torch.zeros(len(at), n, dtype=torch.float64, device="cuda")
  dw = torch.zeros(3, n, k, dtype=torch.float64, device="cuda")
  for i, r in enumerate(at):
    for e, (lo, hi) in enumerate(up.spans(offsets, t)):
      if lo <= r < hi:
        want[i] = w[e].double() @ x[r].double()
        dw[e] += dy[r].double()[:, None] * x[r].double()
  _same(y[at], want)
  y[at] = 0
  assert (y == 0).all()
  _same(ops.grouped_matmul_wgrad(x, dy, offs), dw)
