"""The grouped and 8-bit matrix products without a GPU: the C-ABI of include/cap2det_products.h, its refusals and
those of the wrappers, what a call passes on."""
import ctypes
import os
import re
import subprocess
import threading

import pytest
import torch

from cap2det_amd import _lib
from cap2det_amd import hip_ops as ops

BF16, F32, E4M3, E5M2 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e5m2


# -- library ------------------------------------------------------------------------------------

def test_library_exports_what_the_header_declares():
  lib = _lib.load()
  out = subprocess.check_output(["nm", "-D", "--defined-only", _lib.LIB_PATH]).decode()
  declared = _lib.product_signatures()
  assert set(declared) == set(re.findall(r" T (c2dp_\w+)", out))
  # an entry point more or less is another version
  assert {100: 7}[_lib.product_abi_version()] == len(declared)
  assert lib.c2dp_version() == _lib.product_abi_version()
  text = open(_lib.PRODUCTS_HEADER_PATH).read()
  code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
  assert 'extern "C"' in code
  for banned in ("torch", "at::", "std::", "hipStream_t", "template", "class "):
    assert banned not in code


def test_a_library_of_another_version_is_refused(monkeypatch):
  monkeypatch.setattr(_lib, "_lib", None)
  monkeypatch.setattr(_lib, "product_abi_version", lambda: 99)
  with pytest.raises(ImportError, match="cap2det_products.h"):
    _lib.load()


def test_every_product_can_be_part_of_a_step_plan():
  lib = _lib.load()
  plan = ctypes.c_void_p(lib.c2d_plan_create())
  try:
    for name, (restype, argtypes) in _lib.product_signatures().items():
      if restype is not ctypes.c_int:
        continue
      n = len(argtypes)
      zeros = (ctypes.c_longlong * max(n, 1))(), (ctypes.c_uint8 * max(n, 1))(), (ctypes.c_int * max(n, 1))()
      assert lib.c2d_plan_add_call(plan, name.encode(), n, *zeros) == 0, name
      assert lib.c2d_plan_add_call(plan, name.encode(), n - 1, *zeros) == -1, name
  finally:
    lib.c2d_plan_destroy(plan)


P, ODD, BIG = 4096, 4100, 1 << 23     # addresses that nobody reads: every call here ends on the host


def _quantize(**kw):
  a = dict(x=P, x_type=1, ldx=256, x_batch=0, q=P, q_type=2, scale=P, batch=1, rows=4, cols=256, block_rows=1)
  a.update(kw)
  return _lib.load().c2dp_fp8_quantize(*a.values(), None)


def _fp8(**kw):
  a = dict(a=P, a_type=2, lda=256, a_scale=P, b=P, b_scale=P, offsets=None, groups=1, bias=None, relu=0, y=P, y_type=1,
           ldy=64, rows=4, n=64, k=256, clear=0)
  a.update(kw)
  return _lib.load().c2dp_fp8_matmul(*a.values(), None)


def _rows(dgrad=False, **kw):
  a = dict(x=P, x_type=1, ldx=256, w=P, offsets=P, groups=2, y=P, y_type=1, ldy=256, rows=4, n=256, k=256, clear=0)
  a.update(kw)
  return getattr(_lib.load(), "c2dp_grouped_matmul_dgrad" if dgrad else "c2dp_grouped_matmul")(*a.values(), None)


def _wgrad(**kw):
  a = dict(x=P, x_type=1, ldx=256, dy=P, lddy=64, offsets=P, groups=2, dw=P, rows=4, n=64, k=256, accumulate=0,
           workspace=None, workspace_bytes=0)
  a.update(kw)
  return _lib.load().c2dp_grouped_matmul_wgrad(*a.values(), None)


@pytest.mark.parametrize("call,bad", [
    (_quantize, dict(x=None)), (_quantize, dict(q=None)), (_quantize, dict(scale=None)), (_quantize, dict(x_type=2)),
    (_quantize, dict(q_type=1)), (_quantize, dict(ldx=255)), (_quantize, dict(rows=-1)), (_quantize, dict(cols=-1)),
    (_quantize, dict(batch=-1)), (_quantize, dict(block_rows=64)), (_quantize, dict(block_rows=0)),
    (_fp8, dict(a=None)), (_fp8, dict(a_scale=None)), (_fp8, dict(b=None)), (_fp8, dict(b_scale=None)), (_fp8, dict(y=None)),
    (_fp8, dict(a_type=1)), (_fp8, dict(y_type=2)), (_fp8, dict(lda=255)), (_fp8, dict(ldy=63)), (_fp8, dict(groups=0)),
    (_fp8, dict(groups=2)), (_fp8, dict(rows=-1)), (_fp8, dict(n=-1)), (_fp8, dict(k=-1)),
    (_rows, dict(x=None)), (_rows, dict(w=None)), (_rows, dict(offsets=None)), (_rows, dict(y=None)), (_rows, dict(x_type=2)),
    (_rows, dict(x_type=0, y_type=1)), (_rows, dict(y_type=3)), (_rows, dict(ldx=255)), (_rows, dict(ldy=255)),
    (_rows, dict(groups=0)), (_rows, dict(rows=-1)), (_rows, dict(dgrad=True, n=512)), (_rows, dict(dgrad=True, k=512)),
    (_wgrad, dict(x=None)), (_wgrad, dict(dy=None)), (_wgrad, dict(offsets=None)), (_wgrad, dict(dw=None)),
    (_wgrad, dict(x_type=3)), (_wgrad, dict(ldx=255)), (_wgrad, dict(lddy=63)), (_wgrad, dict(groups=0)), (_wgrad, dict(n=-1)),
], ids=lambda v: "-".join("%s=%s" % p for p in v.items()) if isinstance(v, dict) else v.__name__.strip("_"))
def test_invalid_arguments_end_on_the_host(call, bad):
  assert call(**bad) == -1


def test_unsupported_pitches_and_short_workspaces_end_on_the_host():
  assert _fp8(lda=BIG) == -2 and _rows(ldx=BIG) == -2 and _wgrad(ldx=BIG) == -2 and _wgrad(lddy=BIG) == -2
  assert _rows(x_type=0, y_type=0, ldx=1 << 21) == -2      # (bytes, not elements)
  need = _lib.load().c2dp_grouped_matmul_wgrad_workspace_bytes(1, 8192, 64, 256, 1)
  assert need > 0 and need % (4 * 64 * 256) == 0
  assert _wgrad(groups=1, rows=8192, workspace=P, workspace_bytes=need - 1) == -4
  assert _wgrad(groups=1, rows=8192, workspace=None, workspace_bytes=need) == -4
  assert _wgrad(groups=1, rows=8192, workspace=ODD, workspace_bytes=need) == -1


def test_sizes_that_pass_the_limit_end_on_the_host(calls):
  over = 2 ** 30 + 1
  assert _fp8(rows=over) == -2 and _fp8(n=over, ldy=over) == -2 and _quantize(rows=over) == -2 and _quantize(batch=over) == -2
  assert _rows(rows=over) == -2 and _rows(groups=over) == -2 and _rows(dgrad=True, rows=over) == -2
  assert _wgrad(rows=over) == -2 and _wgrad(groups=over) == -2
  for many in (over, 2 ** 32 + 5):                           # (as 32-bit numbers the latter would be 5 rows)
    x, one = _t(1, 24, dtype=BF16).expand(many, 24), torch.zeros(2, dtype=torch.int32)
    a, s = torch.empty(many, 0, dtype=E4M3), torch.empty(many, 0)
    for f in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_matmul(a, s, _t(8, 0, dtype=E4M3), _t(1, 0)),
              lambda: ops.grouped_matmul_fp8(a, s, _t(1, 8, 0, dtype=E4M3), _t(1, 1, 0), one),
              lambda: ops.grouped_matmul(x, W[:1], one), lambda: ops.grouped_matmul_dgrad(x, _t(1, 24, 8, dtype=BF16), one),
              lambda: ops.grouped_matmul_wgrad(x, x, one)):
      with pytest.raises(ValueError, match="rows, columns and groups up to 1073741824"):
        f()
  assert not calls


def test_empty_calls_are_no_calls():
  for empty in (dict(rows=0), dict(cols=0, ldx=0), dict(batch=0)):
    assert _quantize(x=None, q=None, scale=None, **empty) == 0
  assert _fp8(rows=0, y=None, a=None) == 0 and _fp8(n=0, y=None) == 0
  assert _rows(rows=0, y=None, x=None) == 0 and _rows(n=0, y=None) == 0 and _rows(dgrad=True, k=0, y=None) == 0
  assert _wgrad(n=0, dw=None) == 0 and _wgrad(k=0, dw=None) == 0


def test_workspace_is_nothing_where_tiles_are_many_or_arguments_are_none():
  f = _lib.load().c2dp_grouped_matmul_wgrad_workspace_bytes
  assert f(32, 16384, 2048, 2048, 1) == 0
  assert f(0, 10, 10, 10, 1) == f(1, 0, 10, 10, 1) == f(1, 10, 0, 10, 1) == f(1, 10, 10, 10, 2) == 0
  for rows in (1, 100, 5000, 1 << 20, 2 ** 31 - 1):
    for kind in (0, 1):
      assert f(1, rows, 512, 512, kind) <= 256 << 20


def test_loads_written_as_assembly_wait_for_their_scalar_operands():
  """Five wait states lie between a vector instruction's write of a scalar register and a load's read of it; the compiler
  counts none for a load inside inline assembly, so the block has them: one an instruction, n + 1 of s_nop n."""
  csrc = os.path.join(os.path.dirname(_lib.__file__), "csrc")
  found = 0
  for name in sorted(os.listdir(csrc)):
    if name.endswith((".h", ".hip")):
      with open(os.path.join(csrc, name)) as f:
        blocks = re.findall(r'asm volatile\(((?:\s*"[^"]*")+)', f.read())
      for block in blocks:
        waited = 0
        for line in "".join(re.findall(r'"([^"]*)"', block)).replace("\\t", "").split("\\n"):
          op = line.split()
          if not op:                                         # (a barrier for the compiler alone)
            continue
          if op[0].startswith(("buffer_load", "buffer_store", "global_load", "global_store")):
            found += 1
            assert waited >= 5, (name, block)
          waited += int(op[1]) + 1 if op[0] == "s_nop" else 1
  assert found


# -- wrappers -------------------------------------------------------------------------------------

@pytest.fixture
def calls(monkeypatch):
  """The wrappers as on a device, with CPU tensors: what they pass on instead of the call."""
  seen = []
  monkeypatch.setattr(ops, "_device", lambda: -1)
  monkeypatch.setattr(ops, "_stream", lambda: 0)
  monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name,) + args))
  return seen


def _t(*shape, dtype=F32):
  return torch.zeros(*shape).to(dtype)


def _fp8_args(m=4, n=200, k=272, groups=None):
  lead = () if groups is None else (groups,)
  return dict(a=_t(m, k, dtype=E4M3), a_scale=_t(m, 3), b=_t(*lead, n, k, dtype=E4M3), b_scale=_t(*lead, 2, 3))


OFFS = torch.tensor([0, 2, 4], dtype=torch.int32)


def test_calls_that_are_accepted_and_what_they_pass_on(calls):
  x = _t(4, 300, dtype=BF16)
  q, s = ops.fp8_quantize(x[:, :272], 128, E5M2)
  assert q.shape == (4, 272) and q.dtype == E5M2 and s.shape == (1, 3)
  assert calls.pop() == ("c2dp_fp8_quantize", x.data_ptr(), 1, 300, 0, q.data_ptr(), 3, s.data_ptr(), 1, 4, 272, 128, 0)
  x = _t(5, 4, 272)
  q, s = ops.fp8_quantize(x[::2])
  assert calls.pop() == ("c2dp_fp8_quantize", x.data_ptr(), 0, 272, 2 * 4 * 272, q.data_ptr(), 2, s.data_ptr(), 3, 4, 272, 1, 0)
  v = _fp8_args()
  y = ops.fp8_matmul(**v, relu=True)
  p = {k: t.data_ptr() for k, t in v.items()}
  assert y.dtype == BF16 and y.shape == (4, 200)
  assert calls.pop() == ("c2dp_fp8_matmul", p["a"], 2, 272, p["a_scale"], p["b"], p["b_scale"], None, 1, None, 1,
                         y.data_ptr(), 1, 200, 4, 200, 272, 1, 0)
  v = _fp8_args(groups=2)
  out, bias = _t(4, 256), _t(2, 200)
  y = ops.grouped_matmul_fp8(**v, offsets=OFFS, out=out[:, 8:208], bias=bias)
  assert y.data_ptr() == out.data_ptr() + 32
  got = calls.pop()
  assert got[7:11] == (OFFS.data_ptr(), 2, bias.data_ptr(), 0) and got[11:] == (y.data_ptr(), 0, 256, 4, 200, 272, 0, 0)
  x, w, dy = _t(4, 24, dtype=BF16), _t(2, 16, 24, dtype=BF16), _t(4, 16, dtype=BF16)
  y = ops.grouped_matmul(x, w, OFFS)
  assert calls.pop() == ("c2dp_grouped_matmul", x.data_ptr(), 1, 24, w.data_ptr(), OFFS.data_ptr(), 2, y.data_ptr(), 1, 16,
                         4, 16, 24, 1, 0)
  y = ops.grouped_matmul_dgrad(dy, w, OFFS, out_dtype=F32)
  assert calls.pop() == ("c2dp_grouped_matmul_dgrad", dy.data_ptr(), 1, 16, w.data_ptr(), OFFS.data_ptr(), 2, y.data_ptr(), 0,
                         24, 4, 16, 24, 1, 0)
  dw = ops.grouped_matmul_wgrad(x, dy, OFFS)
  assert dw.shape == (2, 16, 24) and dw.dtype == F32
  assert calls.pop() == ("c2dp_grouped_matmul_wgrad", x.data_ptr(), 1, 24, dy.data_ptr(), 16, OFFS.data_ptr(), 2, dw.data_ptr(),
                         4, 16, 24, 0, None, 0, 0)
  # a row whose pitch says nothing, and nothing to do
  ops.grouped_matmul(x[:1].expand(1, 24), w, OFFS)
  assert calls.pop()[3] == 24
  ops.grouped_matmul(x[:0], w, OFFS)
  ops.fp8_quantize(_t(0, 7))
  assert not calls


def test_a_step_plan_keeps_what_the_calls_that_it_records_allocate(calls, monkeypatch):
  class Recorder(object):
    keep = []
  monkeypatch.setattr(_lib, "recorder", Recorder)
  x, dy = _t(8192, 256, dtype=BF16), _t(8192, 192, dtype=BF16)
  offs = torch.tensor([0, 8192], dtype=torch.int32)
  v, w = _fp8_args(), _t(1, 192, 256, dtype=BF16)

  def run():
    """Addresses that the calls write to."""
    ops.grouped_matmul_wgrad(x, dy, offs, out=torch.zeros(1, 192, 256))
    held = {calls[-1][-3]}
    ops.grouped_matmul_wgrad(x, dy, offs)
    held |= {calls[-1][8], calls[-1][-3]}
    ops.fp8_quantize(x)
    held |= {calls[-1][5], calls[-1][7]}
    ops.fp8_matmul(**v)
    held.add(calls[-1][11])
    for dtype in (BF16, F32):
      ops.grouped_matmul(x, w, offs, out_dtype=dtype)
      held.add(calls[-1][7])
    assert None not in held
    return held

  monkeypatch.setattr(_lib, "recorder_thread", threading.get_ident())
  assert run() == {t.data_ptr() for t in Recorder.keep}
  kept = len(Recorder.keep)
  monkeypatch.setattr(_lib, "recorder_thread", -1)                 # (another thread records)
  run()
  assert len(Recorder.keep) == kept
  calls.clear()


X, W, DY = _t(4, 24, dtype=BF16), _t(2, 16, 24, dtype=BF16), _t(4, 16, dtype=BF16)


@pytest.mark.parametrize("f,what", [
    (lambda: ops.fp8_quantize([1.0]), "x: a tensor"),
    (lambda: ops.fp8_quantize(_t(4)), "x: 2 dimensions"),
    (lambda: ops.fp8_quantize(_t(1, 2, 3, 4)), "x: 2 dimensions"),
    (lambda: ops.fp8_quantize(_t(4, 4, dtype=torch.float16)), "x: one of"),
    (lambda: ops.fp8_quantize(_t(4, 4), 2), "block_rows"),
    (lambda: ops.fp8_quantize(_t(4, 4), 1, BF16), "dtype: one of"),
    (lambda: ops.fp8_quantize(_t(4, 4).t()[:, ::2]), "columns have to be contiguous"),
    (lambda: ops.fp8_quantize(_t(1, 4).expand(3, 4)), "rows overlap"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), a=_t(4, 272))), "a: one of"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), a=_t(4, 271, dtype=E4M3))), "a: 272 columns"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), b=_t(200, 272, dtype=E5M2))), "b: one of"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), b=_t(272, 200, dtype=E4M3).t())), "b: has to be contiguous"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), b=_t(1, 200, 272, dtype=E4M3))), "b: 2 dimensions"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), a_scale=_t(4, 2))), "a_scale: shape"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), a_scale=_t(4, 3, dtype=BF16))), "a_scale: one of"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), a_scale=_t(3, 4).t())), "a_scale: has to be contiguous"),
    (lambda: ops.fp8_matmul(**dict(_fp8_args(), b_scale=_t(200, 3))), "b_scale: shape"),
    (lambda: ops.fp8_matmul(**_fp8_args(), bias=_t(199)), "bias: shape"),
    (lambda: ops.fp8_matmul(**_fp8_args(), bias=_t(200, dtype=BF16)), "bias: one of"),
    (lambda: ops.fp8_matmul(**_fp8_args(), out_dtype=torch.float16), "out_dtype"),
    (lambda: ops.fp8_matmul(**_fp8_args(), out=_t(4, 199)), "out: shape"),
    (lambda: ops.fp8_matmul(**_fp8_args(), out=_t(4, 200, dtype=E4M3)), "out: one of"),
    (lambda: ops.grouped_matmul_fp8(**_fp8_args(groups=2), offsets=OFFS[:2]), "offsets: shape"),
    (lambda: ops.grouped_matmul_fp8(**_fp8_args(groups=2), offsets=OFFS.long()), "offsets: one of"),
    (lambda: ops.grouped_matmul_fp8(**_fp8_args(groups=0), offsets=OFFS[:1]), "at least one group"),
    (lambda: ops.grouped_matmul_fp8(**_fp8_args(groups=2), offsets=OFFS, bias=_t(200)), "bias: 2 dimensions"),
    (lambda: ops.grouped_matmul(X, W.float(), OFFS), "w: one of"),
    (lambda: ops.grouped_matmul(X.half(), W.half(), OFFS), "x: one of"),
    (lambda: ops.grouped_matmul(X[:, :23], W, OFFS), "x: 24 columns"),
    (lambda: ops.grouped_matmul(X, W[0], OFFS), "w: 3 dimensions"),
    (lambda: ops.grouped_matmul(X, W.transpose(1, 2), OFFS), "x: 16 columns|contiguous"),
    (lambda: ops.grouped_matmul(X, W, None), "offsets: a tensor"),
    (lambda: ops.grouped_matmul(X, W, OFFS.tolist()), "offsets: a tensor"),
    (lambda: ops.grouped_matmul(X, W[:0], OFFS[:1]), "at least one group"),
    (lambda: ops.grouped_matmul(X, W, torch.zeros(6, dtype=torch.int32)[::2]), "offsets: has to be contiguous"),
    (lambda: ops.grouped_matmul(X.float(), W.float(), OFFS, out_dtype=BF16), "out_dtype"),
    (lambda: ops.grouped_matmul(X.float(), W.float(), OFFS, out=_t(4, 16, dtype=BF16)), "out: one of"),
    (lambda: ops.grouped_matmul_dgrad(X, W, OFFS), "dy: 16 columns"),
    (lambda: ops.grouped_matmul_dgrad(DY, W, OFFS, out=_t(24, 4, dtype=BF16).t()), "columns have to be contiguous"),
    (lambda: ops.grouped_matmul_dgrad(DY, W, OFFS, out=_t(1, 24, dtype=BF16).expand(4, 24)), "rows overlap"),
    (lambda: ops.grouped_matmul_wgrad(X, DY[:3], OFFS), "dy: 4 rows"),
    (lambda: ops.grouped_matmul_wgrad(X, DY.float(), OFFS), "dy: one of"),
    (lambda: ops.grouped_matmul_wgrad(X, DY, OFFS[:1]), "at least two"),
    (lambda: ops.grouped_matmul_wgrad(X, DY, OFFS, accumulate=True), "accumulate"),
    (lambda: ops.grouped_matmul_wgrad(X, DY, OFFS, out=_t(2, 16, 24, dtype=BF16)), "out: one of"),
    (lambda: ops.grouped_matmul_wgrad(X, DY, OFFS, out=_t(2, 24, 16)), "out: shape"),
    (lambda: ops.grouped_matmul_wgrad(X, DY, OFFS, out=_t(2, 24, 16).transpose(1, 2)), "out: has to be contiguous"),
])
def test_wrappers_name_what_is_wrong(calls, f, what):
  with pytest.raises(ValueError, match=what):
    f()
  assert not calls


def test_a_result_that_shares_memory_with_an_operand_is_refused(calls):
  x = _t(4, 48, dtype=BF16)
  with pytest.raises(ValueError, match="shares memory"):
    ops.grouped_matmul(x[:, :24], W, OFFS, out=x[:, 24:40])       # (interleaved rows: refused with the rest)
  flat = torch.zeros(4 * 24 + 4 * 16, dtype=BF16)
  ops.grouped_matmul(flat[:96].view(4, 24), W, OFFS, out=flat[96:].view(4, 16))
  assert len(calls) == 1
  with pytest.raises(ValueError, match="shares memory"):
    ops.grouped_matmul(flat[:96].view(4, 24), W, OFFS, out=flat[95:159].view(4, 16))


def test_tensors_of_another_device_are_refused(monkeypatch):
  monkeypatch.setattr(ops, "_device", lambda: 0)
  for f in (lambda: ops.fp8_quantize(_t(4, 4)), lambda: ops.fp8_matmul(**_fp8_args()),
            lambda: ops.grouped_matmul_fp8(**_fp8_args(groups=2), offsets=OFFS), lambda: ops.grouped_matmul(X, W, OFFS),
            lambda: ops.grouped_matmul_dgrad(DY, W, OFFS), lambda: ops.grouped_matmul_wgrad(X, DY, OFFS)):
    with pytest.raises(ValueError, match="current device cuda:0"):
      f()


def test_the_cases_that_are_measured_run_in_their_plain_form(monkeypatch):
  """perf/operators.py on the CPU, at small sizes: the plain form against the 64-bit definition."""
  import importlib.util
  path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
  spec = importlib.util.spec_from_file_location("perf_operators", path)
  m = importlib.util.module_from_spec(spec)
  spec.loader.exec_module(m)
  monkeypatch.setattr(m, "DEV", "cpu")
  assert not m.own and len({c["name"] for c in m.listed()}) == len(m.listed())
  small = [dict(op="quantize", m=37, k=208, rows=1, type="bf16", to="e4m3"),
           dict(op="quantize", m=200, k=208, rows=128, type="fp32", to="e5m2"),
           dict(op="fp8", m=37, n=200, k=208, a="e5m2", out="fp32", bias=True),
           dict(op="grouped", way="fwd", t=40, e=7, n=33, k=64, type="fp32", tail=3),
           dict(op="grouped", way="dgrad", t=40, e=50, n=32, k=64, type="fp32", tail=3),
           dict(op="grouped", way="wgrad", t=40, e=7, n=32, k=64, type="fp32", tail=3),
           dict(op="grouped_fp8", t=40, e=7, n=333, k=272, a="e4m3", out="fp32", tail=5)]
  for case in small:
    got, want = m.run(m.prepare(case, 3)), m.exact(case, 3)
    got, want = (v if isinstance(v, dict) else dict(y=v) for v in (got, want))
    for key in got:
      x, y = got[key].double(), want[key]
      assert x.shape == y.shape and (x - y).norm() <= 1e-5 * y.norm(), (case, key)
    w = m.work(case)
    assert w["bytes"] > 0 and w["flops"] > 0
