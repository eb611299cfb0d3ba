"""Inputs and 64-bit oracles of the grouped and 8-bit matrix products."""
import torch

BLOCK = 128


def offsets_of(counts, first=0):
  offs = [first]
  for c in counts:
    offs.append(offs[-1] + c)
  return offs


def spans(offsets, rows):
  """[(lo, hi)] per group: offsets clamped to [0, rows], each at least the largest before it."""
  top, out = 0, []
  clamped = [min(max(o, 0), rows) for o in offsets]
  for a, b in zip(clamped[:-1], clamped[1:]):
    top = max(top, a)
    out.append((top, max(top, b)))
    top = max(top, b)
  return out


def integers(gen, shape, top, dtype=torch.float32, device="cuda"):
  """Whole numbers from -top to top: their products' sums are exact in fp32 while they stay below 2^24."""
  return torch.randint(-top, top + 1, shape, generator=gen, device=device).to(dtype)


def grouped(x, w, offsets):
  """[rows, n] in 64 bits, NaN at rows of no group."""
  y = torch.full((x.shape[0], w.shape[1]), float("nan"), dtype=torch.float64, device=x.device)
  for e, (lo, hi) in enumerate(spans(offsets, x.shape[0])):
    y[lo:hi] = x[lo:hi].double() @ w[e].double().t()
  return y


def grouped_dw(x, dy, offsets):
  groups = len(offsets) - 1
  dw = torch.zeros(groups, dy.shape[1], x.shape[1], dtype=torch.float64, device=x.device)
  for e, (lo, hi) in enumerate(spans(offsets, x.shape[0])):
    dw[e] = dy[lo:hi].double().t() @ x[lo:hi].double()
  return dw


def spread(scale, rows, shape):
  """One scale for each element of [.., m, k], blocks of rows x 128."""
  s = scale.repeat_interleave(BLOCK, -1)[..., :shape[-1]]
  return s.repeat_interleave(rows, -2)[..., :shape[-2], :]


def dequantized(q, scale, rows):
  return q.float().double() * spread(scale.double(), rows, q.shape)


def view_with_pitch(t, pitch, fill, column=0):
  """The same matrix as columns [column, column + cols) of a wider one that holds `fill` elsewhere."""
  big = torch.full((t.shape[0], pitch), fill, dtype=torch.float32, device=t.device).to(t.dtype)
  big[:, column:column + t.shape[1]] = t
  return big[:, column:column + t.shape[1]]


def half_step(dtype):
  """Largest rounding error of a type relative to the value."""
  return torch.finfo(dtype).eps / 2


def sum_bound(terms, abs_sum):
  """Error of a sum of `terms` products in fp32, in any order and with each addition rounded or cut off (2^-23
  relative to the partial sum, which is at most the sum of magnitudes)."""
  return terms * 2.0 ** -23 * abs_sum


def assert_within(got, want, tol, what=""):
  got, want = got.double(), want.double()
  assert torch.isfinite(want).all()
  bad = ~((got - want).abs() <= tol)
  assert not bad.any(), "%s: %d of %d values off, first at %s: %r for %r" % (
      what, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item())
