"""What the grouped and 8-bit products do not take is refused on the host, by name and as a ValueError."""
import pytest
import torch

from cap2det_amd import _lib
from cap2det_amd import hip_ops as ops

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
P = 4096                                     # an address that nobody reads: every call here ends on the host


@pytest.fixture
def host(monkeypatch):
  """The wrappers with CPU tensors: what they pass on would be refused by the library, or fails the test."""
  monkeypatch.setattr(ops, "_device", lambda: -1)
  monkeypatch.setattr(ops, "_stream", lambda: 0)
  monkeypatch.setattr(_lib, "call", lambda name, *args: pytest.fail(name))


def _far(rows, cols, step, dtype):
  """Rows `step` elements apart, of memory that nobody writes."""
  return torch.empty(0, dtype=dtype).set_(torch.empty((rows - 1) * step + cols, dtype=dtype).untyped_storage(), 0, (rows, cols), (step, 1))


OFFS = torch.tensor([0, 1, 2], dtype=torch.int32)
MB4 = 1 << 22


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_too_far_apart_are_named(host, dtype):
  es = 2 if dtype == BF16 else 4
  x, near, w = _far(2, 24, MB4 // es + 1, dtype), torch.zeros(2, 16, dtype=dtype), torch.zeros(2, 16, 24, dtype=dtype)
  got = " 4194304 bytes apart are taken, got %d" % (MB4 + es)
  for f, name in ((lambda: ops.grouped_matmul(x, w, OFFS), "x"), (lambda: ops.grouped_matmul_wgrad(x, near, OFFS), "x"),
                  (lambda: ops.grouped_matmul_wgrad(near, x, OFFS), "dy"),
                  (lambda: ops.grouped_matmul_dgrad(x, torch.zeros(2, 24, 8, dtype=dtype), OFFS), "dy"),
                  (lambda: ops.grouped_matmul(torch.zeros(2, MB4 // es + 1, dtype=dtype), torch.zeros(2, 1, MB4 // es + 1, dtype=dtype), OFFS), "x"),
                  (lambda: ops.grouped_matmul_dgrad(torch.zeros(2, 1, dtype=dtype), torch.zeros(2, 1, MB4 // es + 1, dtype=dtype), OFFS), "w")):
    with pytest.raises(ValueError, match="^%s: rows up to%s" % (name, got)):
      f()


def test_8_bit_rows_too_far_apart_are_named(host):
  a, b = _far(2, 128, MB4 + 1, E4M3), torch.zeros(1, 128).to(E4M3)
  one = torch.ones(2, 1)
  with pytest.raises(ValueError, match="^a: rows up to 4194304 bytes apart are taken, got 4194305"):
    ops.fp8_matmul(a, one, b, one[:1])
  with pytest.raises(ValueError, match="^a: rows up to"):
    ops.grouped_matmul_fp8(a, one, b[None].expand(2, 1, 128).contiguous(), one.view(2, 1, 1), OFFS)
  wide = torch.zeros(2, MB4 + 16, dtype=torch.uint8).view(E4M3)
  scale = torch.ones(2, MB4 // 128 + 1)
  with pytest.raises(ValueError, match="^a: rows up to"):
    ops.fp8_matmul(wide, scale, wide[:1], scale[:1])


def test_rows_at_the_largest_pitch_are_passed_on(monkeypatch):
  seen = []
  monkeypatch.setattr(ops, "_device", lambda: -1)
  monkeypatch.setattr(ops, "_stream", lambda: 0)
  monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(args))
  x, dy = _far(2, 24, MB4 // 2, BF16), torch.zeros(2, 16, dtype=BF16)
  ops.grouped_matmul(x, torch.zeros(2, 16, 24, dtype=BF16), OFFS)
  ops.grouped_matmul_wgrad(x, dy, OFFS)
  ops.fp8_quantize(_far(2, 24, MB4, BF16))                    # (the quantiser takes any)
  assert [a[2] for a in seen] == [MB4 // 2, MB4 // 2, MB4]


def test_many_groups_are_refused(host):
  many = (1 << 16) + 1
  offs = torch.zeros(many + 1, dtype=torch.int32)
  x, w = torch.zeros(2, 8, dtype=BF16), torch.zeros(many, 8, 8, dtype=BF16)
  a, b = torch.zeros(2, 8).to(E4M3), torch.zeros(many, 8, 8, dtype=torch.uint8).view(E4M3)
  for f in (lambda: ops.grouped_matmul(x, w, offs), lambda: ops.grouped_matmul_dgrad(x, w, offs),
            lambda: ops.grouped_matmul_wgrad(x, x, offs),
            lambda: ops.grouped_matmul_fp8(a, torch.ones(2, 1), b, torch.ones(many, 1, 1), offs)):
    with pytest.raises(ValueError, match="up to 65536 groups are taken, got 65537"):
      f()
  lib = _lib.load()
  assert lib.c2dp_grouped_matmul(P, 1, 8, P, P, many, P, 1, 8, 2, 8, 8, 0, None) == -2
  assert lib.c2dp_grouped_matmul_dgrad(P, 1, 8, P, P, many, P, 1, 8, 2, 8, 8, 0, None) == -2
  assert lib.c2dp_grouped_matmul_wgrad(P, 1, 8, P, 8, P, many, P, 2, 8, 8, 0, None, 0, None) == -2
  assert lib.c2dp_fp8_matmul(P, 2, 8, P, P, P, P, many, None, 0, P, 1, 8, 2, 8, 8, 0, None) == -2


def test_what_the_library_does_not_take_is_a_value_error_too():
  """65536 rows in groups of one by 2^24 columns: more tiles than are numbered."""
  with pytest.raises(ValueError, match="c2dp_grouped_matmul failed: .*-2"):
    _lib.call("c2dp_grouped_matmul", P, 1, 1, P, P, 1 << 16, P, 1, 1 << 30, 1 << 16, 1 << 30, 1, 0, None)
  with pytest.raises(_lib.Cap2DetHipError):
    _lib.call("c2dp_fp8_quantize", P, 1, 1 << 30, 0, P, 2, P, 1, 1 << 30, 1 << 30, 128, None)
  with pytest.raises(_lib.Cap2DetHipError) as e:
    _lib.call("c2dp_grouped_matmul", None, 1, 1, P, P, 1, P, 1, 1, 1, 1, 1, 0, None)
  assert not isinstance(e.value, ValueError)
