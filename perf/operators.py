"""What is measured of the low-precision and grouped matrix products (cap2det_amd.hip_ops).

Three operators, as a layer of experts uses them together:

  fp8_quantize            x -> (q, scale): 8-bit values and one fp32 scale for every block of 1 x 128
                          (activations) or 128 x 128 (weights) elements
  fp8_matmul,             y = act(sum over blocks of 128 k of  a_scale * b_scale * (a . b)  + bias), for
  grouped_matmul_fp8      one weight matrix, or for one per group of rows
  grouped_matmul,         y_e = x_e . w_e^T and its two gradients, the rows of x sorted by group
  grouped_matmul_dgrad,   (expert) and the groups of any length, zero among them
  grouped_matmul_wgrad

`own` is false: `run` is the plain form, in fp32 with torch's own operations.  `own` is true: `run` makes
the framework's calls on the same inputs.
"""
import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 128
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
F8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
F8_MANTISSA = {"e4m3": 3, "e5m2": 2}
F8_MIN_EXP = {"e4m3": -6, "e5m2": -14}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp32": 4}


def _blocks(n):
  return -(-n // BLOCK)


def listed():
  return [
      # the activation of one token in front of an 8-bit layer: nothing but latency
      dict(name="quantize_one_row", op="quantize", m=1, k=4096, rows=1, type="bf16", to="e4m3"),
      # the pooled features of one image's 2000 proposals less one, fp32 as the heads get them
      dict(name="quantize_rois", op="quantize", m=1999, k=1024, rows=1, type="fp32", to="e4m3"),
      # the activations of a long prompt or a large batch
      dict(name="quantize_activations", op="quantize", m=32768, k=8192, rows=1, type="bf16", to="e4m3"),
      # a weight matrix after an optimiser step, in square blocks
      dict(name="quantize_weights", op="quantize", m=8192, k=4096, rows=128, type="fp32", to="e4m3"),
      # one token through one layer: the weights are read once and nothing else counts
      dict(name="fp8_one_row", op="fp8", m=1, n=8192, k=4096, a="e4m3", out="bf16", bias=True),
      # the five detection heads of 80 classes as one product over 2000 proposals
      dict(name="fp8_heads", op="fp8", m=2000, n=416, k=1024, a="e4m3", out="fp32", bias=True),
      # a large batch through a large layer: the matrix pipe's own case
      dict(name="fp8_large", op="fp8", m=8192, n=8192, k=8192, a="e4m3", out="bf16", bias=False),
      # eight tokens with eight experts each out of 64: most of the weights, a row or two for each
      dict(name="grouped_few_rows", op="grouped", way="fwd", t=64, e=64, n=2048, k=1024, type="bf16", tail=0),
      # a prompt through a layer of 32 experts
      dict(name="grouped_prompt", op="grouped", way="fwd", t=16384, e=32, n=2048, k=2048, type="bf16", tail=0),
      # the input gradient of a ragged batch that ends in padding rows
      dict(name="grouped_dgrad_ragged", op="grouped", way="dgrad", t=5003, e=8, n=1000, k=1536, type="bf16", tail=117),
      # the weight gradients of the prompt's layer
      dict(name="grouped_wgrad", op="grouped", way="wgrad", t=16384, e=32, n=2048, k=2048, type="bf16", tail=0),
      # the prompt through 64 experts in 8 bits
      dict(name="grouped_fp8_prompt", op="grouped_fp8", t=8192, e=64, n=4096, k=2048, a="e4m3", out="bf16", tail=0),
  ]


def _log(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(("quantize", "fp8", "grouped", "grouped", "grouped_fp8"))
  if op == "quantize":
    rows = rng.choice((1, 1, 128))
    return dict(op=op, m=_log(rng, 1, 16384), k=16 * _log(rng, 4, 512), rows=rows,
                type=rng.choice(("bf16", "fp32")), to=rng.choice(("e4m3", "e4m3", "e5m2")))
  if op == "fp8":
    return dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 100, 8192), k=16 * _log(rng, 8, 512),
                a=rng.choice(("e4m3", "e4m3", "e5m2")), out=rng.choice(("bf16", "bf16", "fp32")),
                bias=rng.random() < 0.5)
  t, e = _log(rng, 1, 16384), _log(rng, 1, 64)
  tail = rng.choice((0, 0, _log(rng, 1, 300)))
  if op == "grouped_fp8":
    return dict(op=op, t=t, e=e, n=_log(rng, 100, 4096), k=16 * _log(rng, 8, 128),
                a=rng.choice(("e4m3", "e4m3", "e5m2")), out=rng.choice(("bf16", "bf16", "fp32")), tail=tail)
  way = rng.choice(("fwd", "dgrad", "wgrad"))
  kind = rng.choice(("bf16", "bf16", "fp32"))
  if kind == "fp32":
    t = min(t, 4096)
  n = _log(rng, 64, 2048) if way == "fwd" else 8 * _log(rng, 8, 256)
  return dict(op=op, way=way, t=t, e=e, n=n, k=8 * _log(rng, 8, 256), type=kind, tail=tail)


# -- inputs ---------------------------------------------------------------------------------

def _gen(seed):
  return torch.Generator(device=DEV).manual_seed(seed)


def _activations(gen, m, k):
  """Normal values under one lognormal factor for each column: some columns are ten times others."""
  col = torch.exp(0.8 * torch.randn(k, generator=gen, device=DEV))
  x = torch.randn(m, k, generator=gen, device=DEV)
  return x.mul_(col)


def _weights(gen, *shape):
  return torch.randn(*shape, generator=gen, device=DEV).mul_(shape[-1] ** -0.5)


def _to_fp8(x, rows, to):
  """The 8-bit operands that a program has in hand: values and scales of [..., m, k]."""
  m, k = x.shape[-2:]
  mb, kb = -(-m // rows), _blocks(k)
  pad = torch.nn.functional.pad(x, (0, kb * BLOCK - k, 0, mb * rows - m))
  v = pad.view(*x.shape[:-2], mb, rows, kb, BLOCK)
  scale = (v.abs().amax(dim=(-3, -1)) / F8_MAX[to]).clamp(min=2.0 ** -126)
  q = (v / scale[..., :, None, :, None]).view(*x.shape[:-2], mb * rows, kb * BLOCK)[..., :m, :k]
  return q.clamp(-F8_MAX[to], F8_MAX[to]).to(F8[to]).contiguous(), scale.contiguous()


def _offsets(seed, t, e):
  """Where each group begins, and the longest group: t rows dealt to e groups of popularity 0.5 to 1.5."""
  g = torch.Generator().manual_seed(seed)
  popularity = 0.5 + torch.rand(e, generator=g)
  counts = torch.bincount(torch.multinomial(popularity, t, replacement=True, generator=g), minlength=e)
  offs = torch.zeros(e + 1, dtype=torch.int32)
  offs[1:] = counts.cumsum(0)
  return offs.to(DEV), int(counts.max())


def prepare(case, seed):
  gen = _gen(seed)
  s = dict(case=case)
  if case["op"] == "quantize":
    x = (_activations if case["rows"] == 1 else _weights)(gen, case["m"], case["k"])
    s["x"] = x.to(TYPES[case["type"]])
  elif case["op"] == "fp8":
    s["a"], s["a_scale"] = _to_fp8(_activations(gen, case["m"], case["k"]), 1, case["a"])
    s["b"], s["b_scale"] = _to_fp8(_weights(gen, case["n"], case["k"]), 128, "e4m3")
    s["bias"] = torch.randn(case["n"], generator=gen, device=DEV) if case["bias"] else None
  else:
    t, e, n, k = case["t"] + case["tail"], case["e"], case["n"], case["k"]
    # (a program that pads knows its longest group on the host)
    s["offsets"], s["longest"] = _offsets(seed, case["t"], e)
    if case["op"] == "grouped_fp8":
      s["a"], s["a_scale"] = _to_fp8(_activations(gen, t, k), 1, case["a"])
      s["b"], s["b_scale"] = _to_fp8(_weights(gen, e, n, k), 128, "e4m3")
    else:
      dtype = TYPES[case["type"]]
      if case["way"] in ("fwd", "wgrad"):
        s["x"] = _activations(gen, t, k).to(dtype)
      if case["way"] in ("dgrad", "wgrad"):
        s["dy"] = torch.randn(t, n, generator=gen, device=DEV).to(dtype)
      if case["way"] in ("fwd", "dgrad"):
        s["w"] = _weights(gen, e, n, k).to(dtype)
  return s


# -- one pass ---------------------------------------------------------------------------------

def _spread(scale, rows, m, k):
  """One scale for each element of [..., m, k]."""
  scale = scale.repeat_interleave(BLOCK, -1)[..., :k]
  return scale.repeat_interleave(rows, -2)[..., :m, :] if rows > 1 else scale


def _slots(offsets, longest, t):
  """The place of each row among the groups' padded rows; rows of no group share one behind them."""
  e = offsets.numel() - 1
  row = torch.arange(t, device=offsets.device)
  offs = offsets.long()
  group = torch.searchsorted(offs[1:].contiguous(), row, right=True)
  at = group.clamp(max=e - 1) * longest + row - offs[group.clamp(max=e - 1)]
  return torch.where(group < e, at, e * longest)


def _pad(x, slot, e, longest):
  out = torch.zeros(e * longest + 1, x.shape[1], device=x.device)
  out[slot] = x.float()
  return out[:-1].view(e, longest, x.shape[1])


def _unpad(y, slot):
  y = y.reshape(-1, y.shape[-1])
  return torch.cat([y, torch.zeros(1, y.shape[1], device=y.device)])[slot]


def _plain(s):
  case = s["case"]
  if case["op"] == "quantize":
    q, scale = _to_fp8(s["x"].float(), case["rows"], case["to"])
    return dict(q=q, scale=scale)
  if case["op"] == "fp8":
    m, n, k = case["m"], case["n"], case["k"]
    a = s["a"].float() * _spread(s["a_scale"], 1, m, k)
    b = s["b"].float() * _spread(s["b_scale"], 128, n, k)
    y = a @ b.t()
    return (y if s["bias"] is None else y + s["bias"]).to(TYPES[case["out"]])
  e, longest = case["e"], s["longest"]
  slot = _slots(s["offsets"], longest, case["t"] + case["tail"])
  if case["op"] == "grouped_fp8":
    a = s["a"].float() * _spread(s["a_scale"], 1, s["a"].shape[0], case["k"])
    b = s["b"].float() * _spread(s["b_scale"], 128, case["n"], case["k"])
    return _unpad(torch.bmm(_pad(a, slot, e, longest), b.transpose(1, 2)), slot).to(TYPES[case["out"]])
  dtype = TYPES[case["type"]]
  if case["way"] == "fwd":
    return _unpad(torch.bmm(_pad(s["x"], slot, e, longest), s["w"].float().transpose(1, 2)), slot).to(dtype)
  if case["way"] == "dgrad":
    return _unpad(torch.bmm(_pad(s["dy"], slot, e, longest), s["w"].float()), slot).to(dtype)
  return torch.bmm(_pad(s["dy"], slot, e, longest).transpose(1, 2), _pad(s["x"], slot, e, longest))


def run(state):
  s = state
  if not own:
    return _plain(s)
  from cap2det_amd import hip_ops as ops
  case = s["case"]
  if case["op"] == "quantize":
    q, scale = ops.fp8_quantize(s["x"], case["rows"], F8[case["to"]])
    return dict(q=q, scale=scale)
  if case["op"] == "fp8":
    return ops.fp8_matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
                          out_dtype=TYPES[case["out"]])
  if case["op"] == "grouped_fp8":
    return ops.grouped_matmul_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], s["offsets"],
                                  out_dtype=TYPES[case["out"]])
  if case["way"] == "fwd":
    return ops.grouped_matmul(s["x"], s["w"], s["offsets"])
  if case["way"] == "dgrad":
    return ops.grouped_matmul_dgrad(s["dy"], s["w"], s["offsets"])
  return ops.grouped_matmul_wgrad(s["x"], s["dy"], s["offsets"])


# -- what a pass cannot do without ----------------------------------------------------------------

def work(case):
  if case["op"] == "quantize":
    m, k = case["m"], case["k"]
    return dict(bytes=m * k * (BYTES[case["type"]] + 1) + 4 * -(-m // case["rows"]) * _blocks(k), flops=4 * m * k)
  n, k = case["n"], case["k"]
  kb, nb = _blocks(k), _blocks(n)
  if case["op"] == "fp8":
    m = case["m"]
    return dict(bytes=m * k + 4 * m * kb + n * k + 4 * nb * kb + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0),
                flops=2 * m * n * k)
  t, e, rows = case["t"], case["e"], case["t"] + case["tail"]
  # the groups that get a row: their weights are read, the others' are not
  live = min(e * (1.0 - (1.0 - 1.0 / e) ** t), t) if e > 1 else 1.0
  if case["op"] == "grouped_fp8":
    return dict(bytes=t * (k + 4 * kb) + live * (n * k + 4 * nb * kb) + rows * n * BYTES[case["out"]], flops=2 * t * n * k)
  es = BYTES[case["type"]]
  if case["way"] == "wgrad":
    return dict(bytes=t * (n + k) * es + 4 * e * n * k, flops=2 * t * n * k)
  read, written = (k, n) if case["way"] == "fwd" else (n, k)
  return dict(bytes=(t * read + live * n * k + rows * written) * es, flops=2 * t * n * k)


# -- the definition in 64 bits ----------------------------------------------------------------------

def _round_fp8(v, to):
  """The nearest 8-bit value, ties to even, of |v| up to the type's largest."""
  exp = torch.frexp(v.abs())[1].double().sub_(1).clamp_(min=F8_MIN_EXP[to])
  step = torch.exp2(exp.sub_(F8_MANTISSA[to]))
  return torch.round(v / step).mul_(step)


def _exact_quantize(x, rows, to):
  m, k = x.shape
  q = torch.zeros(m, k, dtype=torch.float64, device=x.device)
  scale = torch.zeros(-(-m // rows), _blocks(k), dtype=torch.float64, device=x.device)
  for j in range(_blocks(k)):
    part = x[:, j * BLOCK:(j + 1) * BLOCK].double()
    top = part.abs().amax(1)
    if rows > 1:
      top = torch.nn.functional.pad(top, (0, -m % rows)).view(-1, rows).amax(1)
    scale[:, j] = (top / F8_MAX[to]).clamp(min=2.0 ** -126)
    of_row = scale[:, j].repeat_interleave(rows)[:m] if rows > 1 else scale[:, j]
    q[:, j * BLOCK:(j + 1) * BLOCK] = _round_fp8(part / of_row[:, None], to)
  return q, scale


def _exact_fp8(a, a_scale, b, b_scale):
  """a [m, k], b [n, k] with scales for 1 x 128 and 128 x 128: the sum over blocks, one block at a time."""
  m, n = a.shape[0], b.shape[0]
  y = torch.zeros(m, n, dtype=torch.float64, device=a.device)
  for j in range(a_scale.shape[1]):
    pa = a[:, j * BLOCK:(j + 1) * BLOCK].float().double() * a_scale[:, j:j + 1].double()
    of_row = torch.cat([b_scale[i:i + 1, j].double().expand(min(BLOCK, n - i * BLOCK)) for i in range(b_scale.shape[0])])
    y += pa @ (b[:, j * BLOCK:(j + 1) * BLOCK].float().double() * of_row[:, None]).t()
  return y


def exact(case, seed):
  s = prepare(case, seed)
  if case["op"] == "quantize":
    q, scale = _exact_quantize(s["x"], case["rows"], case["to"])
    return dict(q=q, scale=scale)
  if case["op"] == "fp8":
    y = _exact_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"])
    return y if s["bias"] is None else y + s["bias"].double()
  begin = s["offsets"].tolist()
  rows, e, n, k = case["t"] + case["tail"], case["e"], case["n"], case["k"]
  if case["op"] == "grouped" and case["way"] == "wgrad":
    dw = torch.zeros(e, n, k, dtype=torch.float64, device=DEV)
    for g in range(e):
      lo, hi = begin[g], begin[g + 1]
      dw[g] = s["dy"][lo:hi].double().t() @ s["x"][lo:hi].double()
    return dw
  y = torch.zeros(rows, k if case["op"] == "grouped" and case["way"] == "dgrad" else n, dtype=torch.float64, device=DEV)
  for g in range(e):
    lo, hi = begin[g], begin[g + 1]
    if lo == hi:
      continue
    if case["op"] == "grouped_fp8":
      y[lo:hi] = _exact_fp8(s["a"][lo:hi], s["a_scale"][lo:hi], s["b"][g], s["b_scale"][g])
    elif case["way"] == "fwd":
      y[lo:hi] = s["x"][lo:hi].double() @ s["w"][g].double().t()
    else:
      y[lo:hi] = s["dy"][lo:hi].double() @ s["w"][g].double()
  return y
