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
