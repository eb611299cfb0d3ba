"""The grouped and 8-bit matrix products in every tile shape, at sizes that the estimated times choose it for: exact sums of
whole numbers."""
import pytest
import torch

from cap2det_amd import hip_ops as ops
from tests import products_cases as cases
from tests import util_products as up

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def _gen(seed=0):
  return torch.Generator(device="cuda").manual_seed(seed)


def _offs(offsets):
  return torch.tensor(offsets, dtype=torch.int32, device="cuda")


def _fp8_operands(gen, m, n, k, a_type, groups=None):
  lead = () if groups is None else (groups,)
  powers = lambda *shape: torch.exp2(torch.randint(-2, 3, shape, generator=gen, device="cuda").float())
  return (up.integers(gen, (m, k), 4).to(a_type), powers(m, -(-k // 128)),
          up.integers(gen, lead + (n, k), 4).to(E4M3), powers(*lead, -(-n // 128), -(-k // 128)))


def _fp8_want(a, a_s, b, b_s):
  return up.dequantized(a, a_s, 1) @ up.dequantized(b, b_s, 128).t()


# More row tiles than an XCD's round holds, the rest of them made as halves: one group and several, ends of groups inside
# and between the halved tiles
@pytest.mark.parametrize("counts,n,k", [([4500], 4096, 264), ([8400], 2048, 520), ([2600, 0, 2400], 4096, 264), ([4600, 256, 30], 4096, 136)])
def test_a_last_round_of_halves(counts, n, k):
  gen = _gen(41)
  offsets = up.offsets_of(counts)
  t = offsets[-1]
  x = up.integers(gen, (t, k), 4, BF16)
  w, wt = up.integers(gen, (len(counts), n, k), 4, BF16), up.integers(gen, (len(counts), k, n), 4, BF16)
  offs = _offs(offsets)
  assert torch.equal(ops.grouped_matmul(x, w, offs), up.grouped(x, w, offsets).to(BF16))
  assert torch.equal(ops.grouped_matmul_dgrad(x, wt, offs), up.grouped(x, wt.transpose(1, 2), offsets).to(BF16))
  a, a_s, b, b_s = _fp8_operands(gen, t, n, k, E4M3, len(counts))
  got = ops.grouped_matmul_fp8(a, a_s, b, b_s, offs)
  for e, (lo, hi) in enumerate(up.spans(offsets, t)):
    assert torch.equal(got[lo:hi], _fp8_want(a[lo:hi], a_s[lo:hi], b[e], b_s[e]).to(BF16))
  if len(counts) == 1:
    assert torch.equal(ops.fp8_matmul(a, a_s, b[0], b_s[0]), got)


# -- every kernel -----------------------------------------------------------------------------------

def _name(case):
  counts = case[0]
  head = "%d" % counts if isinstance(counts, int) else "%dx%d" % (sum(counts), len(counts))
  return "-".join([head] + ["%d" % v for v in case[1:]])


def _off_by_one(t):
  """The same matrix where 16-byte loads do not fit."""
  return up.view_with_pitch(t, t.shape[1] + 5, float("nan"), 1)


def _lead(counts, bad_offsets):
  offsets = up.offsets_of(counts, first=cases.GAP)
  rows = offsets[-1] + cases.TAIL
  if bad_offsets:                              # (outside, falling, and behind the rows)
    offsets[0] = -7
    offsets[2], offsets[3] = offsets[3], offsets[2]
    offsets[-1] = rows + 1000
  return offsets, rows


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("case", cases.FP8_DENSE, ids=_name)
def test_8_bit_products(case, a_type, aligned):
  m, n, k = case
  gen = _gen(n)
  a, a_s, b, b_s = _fp8_operands(gen, m, n, k, a_type)
  bias = up.integers(gen, (n,), 30)
  want = _fp8_want(a, a_s, b, b_s) + bias.double()
  a = a if aligned else _off_by_one(a)
  for dtype in (BF16, F32):
    assert torch.equal(ops.fp8_matmul(a, a_s, b, b_s, out_dtype=dtype, bias=bias, relu=True), want.clamp(min=0).to(dtype))
    big = torch.full((m, n + 9), 77.0, device="cuda", dtype=dtype)
    ops.fp8_matmul(a, a_s, b, b_s, out=big[:, 3:3 + n], bias=bias)
    assert torch.equal(big[:, 3:3 + n], want.to(dtype))
    big[:, 3:3 + n] = 77.0
    assert (big == 77.0).all()


@pytest.mark.parametrize("bad_offsets", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("case", cases.FP8_GROUPED, ids=_name)
def test_grouped_8_bit_products(case, a_type, aligned, bad_offsets):
  counts, n, k = case
  gen = _gen(n)
  offsets, t = _lead(counts, bad_offsets)
  a, a_s, b, b_s = _fp8_operands(gen, t, n, k, a_type, len(counts))
  bias = up.integers(gen, (len(counts), n), 30)
  want = torch.full((t, n), float("nan"), dtype=torch.float64, device="cuda")
  for e, (lo, hi) in enumerate(up.spans(offsets, t)):
    want[lo:hi] = _fp8_want(a[lo:hi], a_s[lo:hi], b[e], b_s[e]) + bias[e].double()
  rest = want.isnan().any(1)
  a_s[rest] = float("inf")
  a[rest] = torch.full((), float("nan"), device="cuda").to(a_type)
  a = a if aligned else _off_by_one(a)
  offs = _offs(offsets)
  for dtype in (BF16, F32):
    got = ops.grouped_matmul_fp8(a, a_s, b, b_s, offs, out_dtype=dtype, bias=bias, relu=True)
    assert torch.equal(got, want.nan_to_num(0.0).clamp(min=0).to(dtype))
    big = torch.full((t, n + 9), 77.0, device="cuda", dtype=dtype)
    ops.grouped_matmul_fp8(a, a_s, b, b_s, offs, out=big[:, 3:3 + n], bias=bias)
    assert torch.equal(big[:, 3:3 + n], want.nan_to_num(77.0).to(dtype))
    big[:, 3:3 + n] = 77.0
    assert (big == 77.0).all()


@pytest.mark.parametrize("bad_offsets", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", cases.ROWS, ids=_name)
def test_grouped_products_and_input_gradients(case, dtype, aligned, bad_offsets):
  counts, n, k = case
  gen = _gen(n)
  offsets, t = _lead(counts, bad_offsets)
  x = up.integers(gen, (t, k), 4, dtype)
  w = up.integers(gen, (len(counts), n, k), 4, dtype)
  want = up.grouped(x, w, offsets)
  x[want.isnan().any(1)] = float("nan")
  x = x if aligned else _off_by_one(x)
  offs, wt = _offs(offsets), w.transpose(1, 2).contiguous()
  for call, weights in ((ops.grouped_matmul, w), (ops.grouped_matmul_dgrad, wt)):
    for out_dtype in (dtype,) if dtype == F32 else (BF16, F32):
      assert torch.equal(call(x, weights, offs, out_dtype=out_dtype), want.nan_to_num(0.0).to(out_dtype))
      big = torch.full((t, n + 9), 77.0, device="cuda", dtype=out_dtype)
      call(x, weights, offs, out=big[:, 3:3 + n])
      assert torch.equal(big[:, 3:3 + n], want.nan_to_num(77.0).to(out_dtype))
      big[:, 3:3 + n] = 77.0
      assert (big == 77.0).all()


@pytest.mark.parametrize("bad_offsets", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", cases.WGRAD, ids=_name)
def test_grouped_weight_gradients(case, dtype, aligned, bad_offsets):
  counts, n, k = case
  gen = _gen(n)
  offsets, t = _lead(counts, bad_offsets and len(counts) > 2)
  x, dy = up.integers(gen, (t, k), 4, dtype), up.integers(gen, (t, n), 4, dtype)
  inside = torch.zeros(t, dtype=torch.bool, device="cuda")
  for lo, hi in up.spans(offsets, t):
    inside[lo:hi] = True
  want = up.grouped_dw(x, dy, offsets)
  x[~inside], dy[~inside] = float("nan"), float("inf")
  x = x if aligned else _off_by_one(x)
  out = ops.grouped_matmul_wgrad(x, dy, _offs(offsets))
  assert torch.equal(out, want.float())
  ops.grouped_matmul_wgrad(x, dy, _offs(offsets), out=out, accumulate=True)
  assert torch.equal(out, 2 * want.float())
