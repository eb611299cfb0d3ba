"""8-bit block-scaled matrices against 64-bit oracles: the quantiser, the product, the grouped product."""
import pytest
import torch

from cap2det_amd import hip_ops as ops
from tests import util_products as up

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
NAN, INF = float("nan"), float("inf")
MAX = {E4M3: 448.0, E5M2: 57344.0}


def _gen(seed=0):
  return torch.Generator(device="cuda").manual_seed(seed)


def _offs(offsets):
  return torch.tensor(offsets, dtype=torch.int32, device="cuda")


def _nearest(v, to):
  """float64 -> the nearest 8-bit value, ties to even, in one rounding: whole numbers of the value's own step."""
  bits, least = (3, -6) if to == E4M3 else (2, -14)
  exponent = (torch.frexp(v.abs())[1] - 1).clamp(min=least).double()
  step = torch.exp2(exponent - bits)
  return (torch.round(v / step) * step).float().to(to)


def _quantized(x, rows, to):
  """The definition.  The scale is correctly rounded to fp32 (through float64, whose 53 bits are more than twice 24
  and 2: rounding twice is rounding once; torch divides by a number on the GPU through its reciprocal, which
  is not).  x F is exact in float64, so that its quotient by the largest value is a tie just where the true one is: a tie
  has at most 5 bits."""
  m, k = x.shape[-2:]
  mb, kb = -(-m // rows), -(-k // 128)
  v = torch.nn.functional.pad(x.float(), (0, kb * 128 - k, 0, mb * rows - m)).view(*x.shape[:-2], mb, rows, kb, 128)
  top = v.abs().nan_to_num(nan=0.0, posinf=INF).amax(dim=(-3, -1))
  scale = (top.double() / MAX[to]).float().clamp(min=2.0 ** -126)
  by = top.double().clamp(min=MAX[to] * 2.0 ** -126)[..., :, None, :, None]
  q = (v.double() * MAX[to] / by).reshape(*x.shape[:-2], mb * rows, kb * 128)[..., :m, :k]
  return _nearest(q, to), scale


def _bits(t):
  return t.view(torch.uint8)


# -- quantiser --------------------------------------------------------------------------------

@pytest.mark.parametrize("to", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 129), (17, 64), (130, 1000), (128, 128), (5, 8200), (257, 384), (1, 9000),
                                 (2000, 520), (33, 127), (64, 16)])
def test_quantize_is_the_definition_bit_for_bit(to, dtype, rows, m, k):
  gen = _gen(m + k)
  x = (torch.randn(m, k, generator=gen, device="cuda") * torch.exp(3 * torch.randn(m, 1, generator=gen, device="cuda"))).to(dtype)
  q, scale = ops.fp8_quantize(x, rows, to)
  want_q, want_s = _quantized(x, rows, to)
  assert q.dtype == to and q.shape == x.shape and scale.shape == (-(-m // rows), -(-k // 128))
  assert torch.equal(scale, want_s)
  assert torch.equal(_bits(q), _bits(want_q))


@pytest.mark.parametrize("to", [E4M3, E5M2])
@pytest.mark.parametrize("exponent", [-118, -100, -41, -38, 0, 100])
def test_quantize_rounds_once(to, exponent):
  """Values one unit in the last place on either side of a tie, and on ties whose scale is not a number of 24 bits (three
  quarters of the largest value: 21 of the steps), from the least scales to large ones; and millions of random ones."""
  gen = _gen(exponent + 200)
  top = (1 + torch.rand(300, 1, generator=gen, device="cuda")) * 2.0 ** exponent
  ties = (2 * torch.randint(8, 16, (300, 100), generator=gen, device="cuda") + 1) if to == E4M3 else \
         (2 * torch.randint(4, 8, (300, 100), generator=gen, device="cuda") + 1)
  x = (top.double() / 1.75 * ties / 16 * torch.exp2(-torch.randint(0, 5, ties.shape, generator=gen, device="cuda").double())).float()
  x = torch.where(x > top, x / 2, x)
  bits = x.view(torch.int32) + torch.randint(-1, 2, x.shape, generator=gen, device="cuda").int()
  even = (top.to(BF16).float() * 0.75) * torch.exp2(-torch.randint(0, 5, (300, 27), generator=gen, device="cuda").float())
  for v in (torch.cat([bits.view(F32), top, top / 3, -top / 7], 1), torch.cat([even, top.to(BF16).float()], 1),
            torch.randn(4000, 1000, generator=gen, device="cuda") * 2.0 ** exponent):
    for rows in (1, 128):
      q, scale = ops.fp8_quantize(v, rows, to)
      want_q, want_s = _quantized(v, rows, to)
      assert torch.equal(scale, want_s) and torch.equal(_bits(q), _bits(want_q))


@pytest.mark.parametrize("to", [E4M3, E5M2])
def test_quantize_ties_zeros_and_ends_of_the_range(to):
  """Every tie of the type against itself: with the block's largest value F the scale is one, and x is the
  quotient."""
  top = MAX[to]
  values = torch.arange(256, dtype=torch.uint8, device="cuda").view(to).float()
  values = values[values.isfinite()].unique()
  mids = (values[1:] + values[:-1]) / 2
  x = torch.zeros(1, 128 * 8, device="cuda")
  flat = torch.cat([values, mids])
  for b in range(8):
    part = flat[b * 100:(b + 1) * 100]
    x[0, b * 128:b * 128 + part.numel()] = part
    x[0, b * 128 + 127] = top
  q, scale = ops.fp8_quantize(x, 1, to)
  assert (scale == 1).all()
  assert torch.equal(_bits(q), _bits(x.to(to)))
  # scales that are no power of two, and quotients on ties of theirs
  for f in (3.0, 5.0 / 7.0, 1.1, 2.0 ** -100 * 1.3, 2.0 ** 100 * 1.7):
    q, scale = ops.fp8_quantize(x * f, 1, to)
    want_q, want_s = _quantized(x * f, 1, to)
    assert torch.equal(scale, want_s) and torch.equal(_bits(q), _bits(want_q)), f
  # zeros, values whose scale is at its least, the largest fp32
  for v in (0.0, 2.0 ** -149, 2.0 ** -126, 2.0 ** -120, 3.4028234663852886e38, -3.4028234663852886e38):
    x = torch.zeros(2, 200, device="cuda")
    x[1, 3] = v
    x[1, 5] = v / 3
    for rows in (1, 128):
      q, scale = ops.fp8_quantize(x, rows, to)
      want_q, want_s = _quantized(x, rows, to)
      assert torch.equal(scale, want_s), v
      # (the sign of a zero is the quotient's)
      assert torch.equal(q.float(), want_q.float()), v


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_nan_and_infinity(dtype, rows):
  gen = _gen(2)
  x = torch.randn(140, 300, generator=gen, device="cuda").to(dtype)
  clean = ops.fp8_quantize(x, rows)
  x[3, 7] = NAN
  x[130, 140] = INF
  q, scale = ops.fp8_quantize(x, rows)
  same = torch.ones(140, 300, dtype=torch.bool, device="cuda")
  same[3, 7] = False
  same[(130 if rows == 1 else 128):(131 if rows == 1 else 140), 128:256] = False
  # (the NaN replaced a value: its own block's maximum may have been that value, which is not so here)
  assert x[3, :128].float().nan_to_num(0).abs().max() > 1
  assert torch.equal(_bits(q)[same], _bits(clean[0])[same])
  assert q[3, 7].float().isnan()
  block = q[(130 if rows == 1 else 128):(131 if rows == 1 else 140), 128:256].float()
  assert block.isnan().all()
  assert scale[130 if rows == 1 else 1, 1] == INF


def test_quantize_strided_and_stacked():
  gen = _gen(4)
  for dtype in (BF16, F32):
    x = torch.randn(70, 200, generator=gen, device="cuda").to(dtype)
    for pitch, column in ((8, 0), (24, 8), (5, 1)):
      v = up.view_with_pitch(x, 200 + pitch, NAN, column)
      for rows in (1, 128):
        got, want = ops.fp8_quantize(v, rows), ops.fp8_quantize(x, rows)
        assert torch.equal(_bits(got[0]), _bits(want[0])) and torch.equal(got[1], want[1])
    w = torch.randn(3, 200, 264, generator=gen, device="cuda").to(dtype)
    for stack in (w, w[:, 1:150], w[:, :, 3:200], w[::2]):
      for rows in (1, 128):
        q, s = ops.fp8_quantize(stack, rows)
        for e in range(stack.shape[0]):
          qe, se = ops.fp8_quantize(stack[e].contiguous(), rows)
          assert torch.equal(_bits(q[e]), _bits(qe)) and torch.equal(s[e], se)
    # square blocks: the transposed matrix has the transposed values and scales
    q, s = ops.fp8_quantize(w[0], 128)
    qt, st = ops.fp8_quantize(w[0].t().contiguous(), 128)
    assert torch.equal(_bits(q).t(), _bits(qt)) and torch.equal(s.t(), st)
  q, s = ops.fp8_quantize(torch.ones(0, 5, device="cuda"))
  assert q.shape == (0, 5) and s.shape == (0, 1)
  q, s = ops.fp8_quantize(torch.ones(5, 0, device="cuda"))
  assert q.shape == (5, 0) and s.shape == (5, 0)


# -- products -----------------------------------------------------------------------------------

def _powers(gen, shape):
  return torch.exp2(torch.randint(-2, 3, shape, generator=gen, device="cuda").float())


def _operands(gen, m, n, k, a_type, groups=None):
  """Whole numbers and scales that are powers of two: exact sums (below 2^24 quarters of a sixteenth)."""
  lead = () if groups is None else (groups,)
  a, b = up.integers(gen, (m, k), 4).to(a_type), up.integers(gen, lead + (n, k), 4).to(E4M3)
  return (a, _powers(gen, (m, -(-k // 128))), b, _powers(gen, lead + (-(-n // 128), -(-k // 128))))


def _want(a, a_scale, b, b_scale, bias=None, relu=False):
  y = up.dequantized(a, a_scale, 1) @ up.dequantized(b, b_scale, 128).t()
  y = y if bias is None else y + bias.double()
  return y.clamp(min=0) if relu else y


SIZES = [(1, 1, 1), (1, 16, 128), (3, 129, 16), (16, 128, 256), (17, 33, 144), (130, 257, 384), (128, 128, 128), (300, 40, 1000),
         (5, 70, 33), (64, 200, 2048), (33, 1000, 528), (200, 300, 130), (1, 300, 4096), (2, 513, 1552), (40, 96, 8192),
         (257, 512, 640), (513, 260, 256), (4100, 4096, 528), (5800, 2048, 256), (2000, 2000, 264)]


@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_of_integers_are_exact(a_type, m, n, k):
  gen = _gen(m + 7 * n + k)
  a, a_s, b, b_s = _operands(gen, m, n, k, a_type)
  bias = up.integers(gen, (n,), 30)
  for add, relu in ((None, False), (bias, False), (bias, True)):
    want = _want(a, a_s, b, b_s, add, relu)
    for dtype in (BF16, F32):
      got = ops.fp8_matmul(a, a_s, b, b_s, out_dtype=dtype, bias=add, relu=relu)
      assert got.dtype == dtype and torch.equal(got, want.float().to(dtype)), (got.double() - want).abs().max()


@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("n,k", [(40, 128), (129, 272), (200, 1024), (33, 67), (520, 640)])
@pytest.mark.parametrize("counts", [[1], [0, 0, 5, 0], [127, 128, 129], [1] * 70, [300, 0, 1, 17], [2, 0, 0, 31, 64]],
                         ids=lambda c: "x".join(map(str, c[:9])))
def test_grouped_products_of_integers_are_exact(a_type, n, k, counts):
  gen = _gen(n + k)
  offsets = up.offsets_of(counts, first=2)
  t = offsets[-1] + 3
  a, a_s, b, b_s = _operands(gen, t, n, k, a_type, len(counts))
  bias = up.integers(gen, (len(counts), n), 30)
  want = torch.zeros(t, n, dtype=torch.float64, device="cuda")
  for e, (lo, hi) in enumerate(up.spans(offsets, t)):
    want[lo:hi] = _want(a[lo:hi], a_s[lo:hi], b[e], b_s[e], bias[e], True)
  for dtype in (BF16, F32):
    got = ops.grouped_matmul_fp8(a, a_s, b, b_s, _offs(offsets), out_dtype=dtype, bias=bias, relu=True)
    assert torch.equal(got, want.float().to(dtype))
  out = torch.full((t, n), 5.0, device="cuda")
  ops.grouped_matmul_fp8(a, a_s, b, b_s, _offs(offsets), out=out, bias=bias, relu=True)
  want[:2], want[offsets[-1]:] = 5.0, 5.0
  assert torch.equal(out, want.float())


def test_large_grouped_tiles_of_integers_are_exact():
  """256 x 256 tiles over ragged groups: last tiles short and long, and a last round that is made as halves."""
  gen = _gen(31)
  for counts, n, k in (([3000, 100, 5900, 0, 256], 2048, 400), ([5800], 2048, 512), ([700, 130, 385] * 8, 4096, 256)):
    offsets = up.offsets_of(counts)
    a, a_s, b, b_s = _operands(gen, offsets[-1], n, k, E4M3, len(counts))
    got = ops.grouped_matmul_fp8(a, a_s, b, b_s, _offs(offsets))
    for e, (lo, hi) in enumerate(up.spans(offsets, offsets[-1])):
      assert torch.equal(got[lo:hi], _want(a[lo:hi], a_s[lo:hi], b[e], b_s[e]).to(BF16))


@pytest.mark.parametrize("a_type", [E4M3, E5M2])
@pytest.mark.parametrize("m,n,k", [(1, 500, 4096), (7, 300, 1000), (40, 1000, 2048), (333, 416, 1024), (1000, 520, 784)])
def test_real_values_within_the_rounding_of_sums(a_type, m, n, k):
  """As a layer uses them: quantise, multiply.  A block's sum of 128 products, its product with a rounded scale, and
  the sum over blocks."""
  gen = _gen(m)
  x = torch.randn(m, k, generator=gen, device="cuda").to(BF16)
  w = torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5
  a, a_s = ops.fp8_quantize(x, 1, a_type)
  b, b_s = ops.fp8_quantize(w, 128)
  da, db = up.dequantized(a, a_s, 1), up.dequantized(b, b_s, 128)
  want, mag = da @ db.t(), da.abs() @ db.abs().t()
  tol = up.sum_bound(min(k, 128) + -(-k // 128) + 2, mag)
  up.assert_within(ops.fp8_matmul(a, a_s, b, b_s, out_dtype=F32), want, tol)
  up.assert_within(ops.fp8_matmul(a, a_s, b, b_s), want, tol + up.half_step(BF16) * (want.abs() + tol))


def test_pitches_garbage_beside_columns_and_bad_values():
  gen = _gen(5)
  m, n, k = 70, 200, 272
  a, a_s, b, b_s = _operands(gen, m, n, k, E4M3)
  want = _want(a, a_s, b, b_s)
  for pitch, column in ((16, 0), (32, 16), (5, 1)):
    av = up.view_with_pitch(a, k + pitch, NAN, column)
    big = torch.full((m, n + pitch), 77.0, device="cuda", dtype=BF16)
    got = ops.fp8_matmul(av, a_s, b, b_s, out=big[:, column:column + n])
    assert torch.equal(got, want.to(BF16))
    big[:, column:column + n] = 77.0
    assert (big == 77.0).all()
  # a NaN value or scale of a row stays in its row, of a weight in its column
  bad = a.clone()
  bad[3, 5] = NAN
  bad_s = a_s.clone()
  bad_s[9, 1] = INF
  got = ops.fp8_matmul(bad, bad_s, b, b_s, out_dtype=F32)
  keep = [i for i in range(m) if i not in (3, 9)]
  assert torch.equal(got[keep], want[keep].float()) and got[3].isnan().all() and not got[9].isfinite().any()
  wbad = b.clone()
  wbad[130, 271] = NAN
  got = ops.fp8_matmul(a, a_s, wbad, b_s, out_dtype=F32, relu=True)
  assert got[:, 130].isnan().all() and torch.equal(got[:, :130], want[:, :130].clamp(min=0).float())


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(9, 200, 272), (130, 200, 400), (1000, 1000, 1100), (1900, 1900, 272), (4000, 4096, 272)])
def test_zero_and_infinite_scales(m, n, k, out_dtype):
  """0 * infinity is a NaN in every kernel; the scales of other rows and columns have no part in it."""
  gen = _gen(m)
  a, a_s, b, b_s = _operands(gen, m, n, k, E4M3)
  a_s[5, 1] = a_s[8, -1] = INF
  b_s[0, 1] = 0.0
  got = ops.fp8_matmul(a, a_s, b, b_s, out_dtype=out_dtype)
  assert got[5, :128].isnan().all() and not got[5].isfinite().any() and not got[8].isfinite().any()
  a_s[5, 1] = a_s[8, -1] = 0.0
  want = _want(a, a_s, b, b_s).to(out_dtype)
  keep = torch.ones(m, dtype=torch.bool, device="cuda")
  keep[5] = keep[8] = False
  assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("m,n,k", [(0, 5, 16), (5, 0, 16), (5, 7, 0)])
def test_empty_sizes(m, n, k):
  a, b = torch.ones(m, k, device="cuda").to(E4M3), torch.ones(n, k, device="cuda").to(E4M3)
  a_s, b_s = torch.ones(m, -(-k // 128), device="cuda"), torch.ones(-(-n // 128), -(-k // 128), device="cuda")
  bias = torch.arange(n, device="cuda").float()
  y = ops.fp8_matmul(a, a_s, b, b_s, bias=bias)
  assert torch.equal(y, bias.to(BF16).expand(m, n))


def test_a_layer_forward_and_input_gradient_with_transposed_weights():
  """dx = dy . w through the same product on w^T, gradients in the wider-ranged 8-bit type."""
  gen = _gen(6)
  m, n, k = 300, 264, 392
  dy = torch.randn(m, n, generator=gen, device="cuda").to(BF16)
  w = torch.randn(n, k, generator=gen, device="cuda") * n ** -0.5
  q, s = ops.fp8_quantize(w, 128)
  g, g_s = ops.fp8_quantize(dy, 1, E5M2)
  dx = ops.fp8_matmul(g, g_s, q.t().contiguous(), s.t().contiguous(), out_dtype=F32)
  dg, dq = up.dequantized(g, g_s, 1), up.dequantized(q, s, 128)
  up.assert_within(dx, dg @ dq, up.sum_bound(128 + 3 + 2, dg.abs() @ dq.abs()))


def test_experts_in_8_bits_and_their_gradients_as_they_run_together():
  """Rows grouped by expert: quantise, up-projection with its activation, quantise, down-projection; the backward pass
  in bf16 on the same offsets; all of it also captured and replayed with other inputs."""
  gen = _gen(7)
  offsets = up.offsets_of([40, 0, 200, 13])
  t, d, h = 253, 256, 320
  offs = _offs(offsets)
  x = torch.randn(t, d, generator=gen, device="cuda").to(BF16)
  dy = torch.randn(t, d, generator=gen, device="cuda").to(BF16)
  w1, w2 = (torch.randn(4, *s, generator=gen, device="cuda") * s[-1] ** -0.5 for s in ((h, d), (d, h)))
  q1, q2 = ops.fp8_quantize(w1, 128), ops.fp8_quantize(w2, 128)
  b1, b2 = w1.to(BF16), w2.to(BF16)

  def layer():
    xa = ops.fp8_quantize(x)
    u = ops.grouped_matmul_fp8(*xa, *q1, offs, relu=True)
    ua = ops.fp8_quantize(u)
    y = ops.grouped_matmul_fp8(*ua, *q2, offs, out_dtype=F32)
    du = ops.grouped_matmul_dgrad(dy, b2, offs) * (u > 0)
    return (y, u, ops.grouped_matmul_dgrad(du, b1, offs, out_dtype=F32), ops.grouped_matmul_wgrad(u, dy, offs),
            ops.grouped_matmul_wgrad(x, du, offs), *xa, *ua, du)

  def check(got):
    y, u, dx, dw2, dw1, xq, xs, uq, us, du = got
    dq1, dq2 = up.dequantized(*q1, 128), up.dequantized(*q2, 128)
    for a, s, dq, out, relu in ((xq, xs, dq1, u, True), (uq, us, dq2, y, False)):
      da = up.dequantized(a, s, 1)
      want, mag = up.grouped(da, dq, offsets), up.grouped(da.abs(), dq.abs(), offsets)
      tol = up.sum_bound(128 + 3 + 2, mag)
      tol = tol + (up.half_step(BF16) * (want.abs() + tol) if out.dtype == BF16 else 0)
      up.assert_within(out, want.clamp(min=0) if relu else want, tol)
    up.assert_within(dx, up.grouped(du, b1.transpose(1, 2), offsets),
                     up.sum_bound(h, up.grouped(du.abs(), b1.abs().transpose(1, 2), offsets)))
    for a, g, out in ((u, dy, dw2), (x, du, dw1)):
      up.assert_within(out, up.grouped_dw(a, g, offsets), up.sum_bound(200, up.grouped_dw(a.abs(), g.abs(), offsets)))

  check(layer())
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = layer()
  for _ in range(3):
    x.copy_(torch.randn(t, d, generator=gen, device="cuda"))
    dy.copy_(torch.randn(t, d, generator=gen, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    check(got)
    for a, b in zip(got, layer()):
      assert torch.equal(a.float(), b.float())


def test_rows_and_weights_behind_four_gigabytes():
  """b is 4.8 GB in 12 groups; the last group's weights and the last rows of a count."""
  groups, n, k = 12, 200000, 2000
  free = torch.cuda.mem_get_info()[0]
  if free < 40 << 30:
    pytest.skip("needs 40 GB")
  gen = _gen(8)
  b = torch.zeros(groups, n, k, device="cuda", dtype=torch.uint8).view(E4M3)
  at = [0, 127, 128, 100001, 199999]
  values = up.integers(gen, (len(at), k), 4).to(E4M3)
  for e in (0, 5, 11):
    b[e].view(torch.uint8)[at] = values.view(torch.uint8)
  b_s = torch.ones(groups, -(-n // 128), 16, device="cuda")
  counts = [1, 0, 0, 0, 0, 3, 0, 0, 0, 0, 0, 20]
  a = up.integers(gen, (24, k), 4).to(E4M3)
  y = ops.grouped_matmul_fp8(a, torch.ones(24, 16, device="cuda"), b, b_s, _offs(up.offsets_of(counts)), out_dtype=F32)
  want = a.float().double() @ values.float().double().t()
  assert torch.equal(y[:, at], want.float())
  y[:, at] = 0
  assert (y == 0).all()
