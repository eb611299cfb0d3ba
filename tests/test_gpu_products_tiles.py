"""The grouped and 8-bit matrix products in every tile shape, at sizes that the estimated times choose it for: exact sums of
whole numbers."""
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
