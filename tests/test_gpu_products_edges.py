"""The grouped and 8-bit matrix products where magnitudes, sizes and arguments are at their ends."""
import pytest
import torch

from cap2det_amd import hip_ops as ops
from tests import util_products as up

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def _gen(seed=0):
  return torch.Generator(device="cuda").manual_seed(seed)


def _offs(offsets):
  return torch.tensor(offsets, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(64, 256), (65, 131), (3, 5)])
def test_a_large_start_keeps_the_shares_of_a_split_gradient(dtype, n, k):
  """A gradient of 8192 ones is added to 2^34, whose step is 2048: the shares of a few hundred rows are each below half
  a step, their sum is four steps.  One rounding: that of start + gradient."""
  rows = 8192
  nbytes = ops._wgrad_workspace_bytes(1, rows, n, k, 1 if dtype == BF16 else 0)
  assert rows * 4 * n * k / nbytes < 1024                   # (rows a share)
  x, dy = torch.ones(rows, k, device="cuda", dtype=dtype), torch.ones(rows, n, device="cuda", dtype=dtype)
  start = torch.full((1, n, k), 2.0 ** 34, device="cuda")
  start[0, ::2] *= -3
  out = start.clone()
  ops.grouped_matmul_wgrad(x, dy, _offs([0, rows]), out=out, accumulate=True)
  assert torch.equal(out, (start.double() + rows).float())


def _cut(a, b, least_a):
  """sum over each 8 k of what the header allows to be lost: 7 * 2^-13 of the largest max(|a|, t) max(|b|, 2^-6)."""
  k = a.shape[1]
  lost = torch.zeros(a.shape[0], b.shape[0], device="cuda")
  for g in range(0, k, 8):
    top = torch.zeros_like(lost)
    for i in range(g, min(g + 8, k)):
      p = a[:, i, None].abs().clamp(min=least_a) * b[None, :, i].abs().clamp(min=2.0 ** -6)
      top = torch.maximum(top, torch.where((a[:, i, None] != 0) & (b[None, :, i] != 0), p, 0.0))
    lost += 7 * 2.0 ** -13 * top
  return lost


# (16 rows and 32 rows from registers; 64, 128 and 256 square tiles)
@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("m,n,k", [(9, 96, 256), (60, 96, 256), (300, 2000, 264), (2000, 2000, 144), (4096, 4096, 256)])
def test_small_products_beside_large_ones_that_cancel(a_type, m, n, k):
  """In every 8 k two large products cancel, or a denormal factor meets a large one, and six small ones are left.  A bf16
  result loses what the header says or less, an fp32 result what fp32 sums lose."""
  gen = _gen(m + k)
  rand = lambda lo, hi, *shape: torch.exp2(torch.randint(lo, hi + 1, shape, generator=gen, device="cuda").float()) * (
      1 + torch.randint(0, 4, shape, generator=gen, device="cuda") / 4) * (1 - 2 * torch.randint(0, 2, shape, generator=gen, device="cuda"))
  a, b = rand(-6, -1, m, k), rand(-6, -1, n, k)
  a[:, 0::8] = rand(5, 7, m, a[:, 0::8].shape[1])
  b[:, 0::8] = rand(4, 7, n, b[:, 0::8].shape[1])
  a[:, 1::8], b[:, 1::8] = a[:, 0::8], -b[:, 0::8]
  a[:, 8:10] = 2.0 ** -9                                      # (denormal in E4M3)
  a[:, 10:16] = rand(-6, -5, m, 6)
  a, b = a.to(a_type), b.to(E4M3)
  a_s, b_s = (torch.exp2(torch.randint(-2, 3, s, generator=gen, device="cuda").float()) for s in ((m, -(-k // 128)), (-(-n // 128), -(-k // 128))))
  da, db = up.dequantized(a, a_s, 1), up.dequantized(b, b_s, 128)
  want = da @ db.t()
  tol = up.sum_bound(128 + -(-k // 128) + 2, da.abs() @ db.abs().t())
  up.assert_within(ops.fp8_matmul(a, a_s, b, b_s, out_dtype=F32), want, tol)
  for c in range(-(-k // 128)):
    at = slice(128 * c, min(128 * c + 128, k))
    tol = tol + _cut(a.float()[:, at], b.float()[:, at], 2.0 ** (-6 if a_type == E4M3 else -14)) * a_s[:, c, None] * up.spread(
        b_s[:, c, None].expand(-1, 1), 128, (n, 1)).t()
  up.assert_within(ops.fp8_matmul(a, a_s, b, b_s), want, tol + up.half_step(BF16) * (want.abs() + tol))


# Sizes whose workgroups, along one dimension of a launch, are more than it holds

@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_stacks_of_many_matrices(rows):
  gen = _gen(51)
  x = torch.randn(70000, 8, 64, generator=gen, device="cuda").to(BF16)
  q, s = ops.fp8_quantize(x, rows)
  want_q, want_s = ops.fp8_quantize(x.view(-1, 64))
  if rows == 1:
    assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8).view(x.shape)) and torch.equal(s, want_s.view(s.shape))
  else:
    assert torch.equal(s, want_s.view(70000, 8, 1).amax(1, keepdim=True))
    for e in (0, 65534, 65535, 69999):
      assert torch.equal(q[e].view(torch.uint8), ops.fp8_quantize(x[e], 128)[0].view(torch.uint8))


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("m,k", [((1 << 30) - 77, 1), (1, 600000007)])
def test_quantize_long_and_wide_matrices(rows, m, k):
  """2^30 rows of one column; more column blocks of a row than a launch has workgroups along y.  Values +-1 and, now and
  then, 2: a block's largest is 1 or 2, 448 or 224 its ones."""
  if torch.cuda.mem_get_info()[0] < 60 << 30:
    pytest.skip("needs 60 GB")
  x = torch.ones(m, k, device="cuda", dtype=BF16)
  flat = x.view(-1)
  flat[::3] = -1
  flat[7::100003] = 2
  q, s = ops.fp8_quantize(x, rows)
  of_scale = 128 if k > 1 else rows                          # elements along the long side that share a scale
  n = flat.numel()
  whole = n // of_scale * of_scale
  top = flat[:whole].view(-1, of_scale).abs().amax(1).float()
  if whole < n:
    top = torch.cat([top, flat[whole:].abs().amax().float()[None]])
  assert torch.equal(s.view(-1), (top.double() / 448).float())
  for lo in range(0, n, of_scale << 20):
    part = flat[lo:lo + (of_scale << 20)].float()
    share = top[lo // of_scale:][:-(-part.numel() // of_scale)].repeat_interleave(of_scale)[:part.numel()]
    got = q.view(torch.uint8).view(-1)[lo:lo + part.numel()].view(E4M3).float()
    assert torch.equal(got, part * 448 / share), lo


def test_products_of_more_row_tiles_than_a_launch_has_along_x():
  """2^28 rows: 2^23 and 2^22 tiles and some.  Every row is one of eight, each result row one of eight."""
  if torch.cuda.mem_get_info()[0] < 60 << 30:
    pytest.skip("needs 60 GB")
  gen = _gen(52)
  t, n, k = (1 << 28) + 1000, 16, 16
  offsets = [3, (1 << 27) + 5, (1 << 27) + 5, t - 50]
  few = up.integers(gen, (8, k), 4, BF16)
  w = up.integers(gen, (3, n, k), 4, BF16)
  x = few.repeat(t // 8, 1)
  offs = _offs(offsets)

  def check(y, want_of):
    assert (y[:3] == 0).all() and (y[t - 50:] == 0).all()
    for e, (lo, hi) in enumerate(up.spans(offsets, t)):
      for at in range(lo, hi, 1 << 25):
        part = y[at:min(hi, at + (1 << 25))]
        want = want_of(e).roll(-(at % 8), 0)
        whole = part.shape[0] // 8 * 8
        assert (part[:whole].view(-1, 8, part.shape[1]) == want).all() and (part[whole:] == want[:part.shape[0] - whole]).all()

  exact = lambda a, b: (a.double() @ b.double()).to(BF16)
  check(ops.grouped_matmul(x, w, offs), lambda e: exact(few, w[e].t()))
  check(ops.grouped_matmul_dgrad(x, w, offs), lambda e: exact(few, w[e]))
  at = torch.tensor([0, 2, 3, 4, 1000003, offsets[1] - 1, offsets[1], (1 << 27) + 6, t - 51, t - 50], device="cuda")
  dy = torch.zeros(t, 8, device="cuda", dtype=BF16)
  dy[at] = up.integers(gen, (len(at), 8), 4, BF16)
  dw = torch.zeros(3, 8, k, dtype=torch.float64, device="cuda")
  for r in at.tolist():
    for e, (lo, hi) in enumerate(up.spans(offsets, t)):
      if lo <= r < hi:
        dw[e] += dy[r].double()[:, None] * x[r].double()
  assert torch.equal(ops.grouped_matmul_wgrad(x, dy, offs), dw.float())
  q, s = x.to(E4M3), torch.ones(t, 1, device="cuda")
  check(ops.grouped_matmul_fp8(q, s, w.to(E4M3), torch.ones(3, 1, 1, device="cuda"), offs), lambda e: exact(few, w[e].t()))


def test_as_many_groups_as_are_taken():
  """65536 groups of no row, one and two, in the forward product's small tiles, its gradients' and the 8-bit product's."""
  gen = _gen(53)
  groups, n, k = 1 << 16, 16, 24
  counts = torch.randint(0, 3, (groups,), generator=gen, device="cuda")
  offs = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
  offs[1:] = counts.cumsum(0)
  t = int(offs[-1])
  of = torch.arange(groups, device="cuda").repeat_interleave(counts)
  x, dy = up.integers(gen, (t, k), 4, BF16), up.integers(gen, (t, n), 4, BF16)
  w = up.integers(gen, (groups, n, k), 4, BF16)
  assert torch.equal(ops.grouped_matmul(x, w, offs), (w[of].float() * x[:, None].float()).sum(-1).to(BF16))
  assert torch.equal(ops.grouped_matmul_dgrad(dy, w, offs), (w[of].float() * dy[:, :, None].float()).sum(1).to(BF16))
  want = torch.zeros(groups, n, k, device="cuda").index_add_(0, of, dy[:, :, None].float() * x[:, None].float())
  assert torch.equal(ops.grouped_matmul_wgrad(x, dy, offs), want)
  y = ops.grouped_matmul_fp8(x.to(E4M3), torch.ones(t, 1, device="cuda"), w.to(E4M3), torch.ones(groups, 1, 1, device="cuda"), offs)
  assert torch.equal(y, (w[of].float() * x[:, None].float()).sum(-1).to(BF16))


def test_the_input_gradient_of_experts_in_8_bits_with_transposed_weights():
  """dx_e = dy_e . w_e through the grouped product on each w_e^T: square blocks transpose with their matrix."""
  gen = _gen(54)
  offsets = up.offsets_of([70, 0, 300, 1])
  t, n, k = offsets[-1], 264, 392
  dy = torch.randn(t, n, generator=gen, device="cuda").to(BF16)
  w = torch.randn(4, n, k, generator=gen, device="cuda") * n ** -0.5
  q, s = ops.fp8_quantize(w, 128)
  g, g_s = ops.fp8_quantize(dy, 1, E5M2)
  qt, st = q.transpose(1, 2).contiguous(), s.transpose(1, 2).contiguous()
  assert torch.equal(qt.view(torch.uint8), ops.fp8_quantize(w.transpose(1, 2).contiguous(), 128)[0].view(torch.uint8))
  dx = ops.grouped_matmul_fp8(g, g_s, qt, st, _offs(offsets), out_dtype=F32)
  dg, dw = up.dequantized(g, g_s, 1), up.dequantized(q, s, 128).transpose(1, 2)
  up.assert_within(dx, up.grouped(dg, dw, offsets), up.sum_bound(128 + 3 + 2, up.grouped(dg.abs(), dw.abs(), offsets)))
