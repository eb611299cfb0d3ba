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
