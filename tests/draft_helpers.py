"""The operators of a step of drafted tokens in 64 bits, for the tests."""

import math

import torch

from tests import fp8_helpers

EPS = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a step, relative to the value


def normed(x, residual, weight, offset, eps, residual_type):
  """(h, out) of the residual norm; h is rounded to residual_type by definition."""
  h = x.double() if residual is None else (x.double() + residual.double()).float().to(residual_type).double()
  y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
  return h, y if weight is None else y * (offset + weight.double())


def eight_bits(y, got, scale):
  """Whether the 8-bit values `got` and scales are those of y, each within its rounding and the slack of y's own."""
  slack = 2.0**-18
  rows, k = y.shape
  for b in range(scale.shape[1]):
    part, q = y[:, b * 128 : (b + 1) * 128], got[:, b * 128 : (b + 1) * 128]
    largest = part.abs().amax(1).clamp(min=2.0**-96)
    assert bool(((scale[:, b] - largest / 448).abs() <= slack * largest / 448).all())
    v = part * (448 / largest)[:, None]
    assert bool(((q - v).abs() <= (2.0**-4 + slack) * v.abs() + 2.0**-10).all())


def rotated(x, pos, freq, amplitude, half):
  """x [rows, heads, dim] in 64 bits."""
  out = x.double().clone()
  pairs = len(freq)
  t = pos.double()[:, None] * freq
  c, s = (amplitude * torch.cos(t))[:, None], (amplitude * torch.sin(t))[:, None]
  first = torch.arange(pairs) if half else 2 * torch.arange(pairs)
  second = first + (pairs if half else 1)
  a, b = x[..., first].double(), x[..., second].double()
  out[..., first], out[..., second] = a * c - b * s, a * s + b * c
  return out


def attention(q, k_pages, v_pages, row0, lengths, page_map, heads, scale, softcap=0.0):
  """(out, bound) [rows, heads, dim] in 64 bits on the inputs' device; rows that see nothing are NaN.  The bound counts probabilities and results rounded to bfloat16
  (half a step of each), scores and sums in 32 bits, and weights off by 2^-13.2 each (2^-12.2 of a quotient of their sums, inside the 2^-12)."""
  kv, num_pages, page, dim = k_pages.shape
  out = torch.full((q.shape[0], heads, dim), math.nan, dtype=torch.float64, device=q.device)
  bound = torch.zeros_like(out)
  for s in range(len(lengths)):
    n = row0[s + 1] - row0[s]
    size = min(lengths[s], page_map.shape[1] * page)
    if n == 0 or size <= 0:
      continue
    pages = page_map[s, : -(-size // page)].long()
    pages = torch.where((pages >= 0) & (pages < num_pages), pages, 0)
    for i in range(n):
      seen = min(lengths[s] - n + i + 1, size)
      if seen <= 0:
        continue
      row = row0[s] + i
      for g in range(kv):
        k = k_pages[g, pages].reshape(-1, dim)[:seen].double()
        v = v_pages[g, pages].reshape(-1, dim)[:seen].double()
        a = slice(g * heads // kv, (g + 1) * heads // kv)
        x = q[row].view(heads, dim)[a].double()
        score = x @ k.T * scale
        off = 2.0**-20 * scale * float((x.abs() @ k.abs().T).max())
        if softcap > 0:
          score = softcap * torch.tanh(score / softcap)
          off += 2.0**-20 * softcap
        p = torch.softmax(score, 1)
        out[row, a] = p @ v
        bound[row, a] = (2.0**-8 + 2 * off + 2.0**-12) * (p @ v.abs()) + 2.0**-8 * out[row, a].abs()
  return out, bound


def counted(l):
  """A logit as it counts."""
  l = torch.where(l.isnan(), -math.inf, l.double())
  return l.clamp(max=float(torch.finfo(torch.float32).max))


def verified(target, draft, row0, token, heat, draft_heat, accept, pick, vocab, close=2.0**-19):
  """Per sequence (accepted, [emitted], whether a draft's fate lies closer to its border than 32-bit weights tell, the tokens that may be the drawn one within their rounding: the first and
  the last).  A weight exp2(x) of a 32-bit x is off by |x| ln 2 2^-24 + 2^-22 at most: what
  counts in a sum has |x| up to 17 or so, 2^-20.5.  Sums of weights that are all off to one side, and the whole sum to the other, are off by 2^-19.5 of it; a probability by
  twice that, and two of them are compared."""
  out = []
  for s in range(len(row0) - 1):
    emitted, near, kept, may = [], False, 0, (-1, -1)
    for r in range(row0[s], row0[s + 1]):
      final = r + 1 == row0[s + 1]
      l = counted(target[r, :vocab])
      x = -1 if final else int(token[r + 1])
      known = 0 <= x < vocab
      empty = bool(l.max() == -math.inf)
      if heat[s] == 0:
        best = -1 if empty else int((l == l.max()).nonzero()[0, 0])
        keep, drawn = not final and known and best == x, best
        may = best, best
      else:
        p = torch.zeros_like(l) if empty else torch.softmax((l - l.max()) / heat[s], 0)
        sure = draft is None or draft_heat[s] == 0
        q = None
        if not final and not sure:
          d = counted(draft[r, :vocab])
          q = torch.zeros_like(d) if bool(d.max() == -math.inf) else torch.softmax((d - d.max()) / draft_heat[s], 0)
        keep = False
        if not final and known:
          left, right = float(accept[r]) * (1.0 if sure else float(q[x])), float(p[x])
          keep = left < right
          near |= left != right and abs(left - right) <= 4 * close * right
        weight = p.clone()
        if not final and sure and known:
          weight[x] = 0
        elif not final and not sure:
          weight = (p - q).clamp(min=0)
        if float(weight.sum()) == 0:
          weight = p
        up = weight.cumsum(0)
        if float(up[-1]) == 0:
          drawn, may = -1, (-1, -1)
        else:
          want, last = float(pick[s]) * float(up[-1]), int(weight.nonzero()[-1, 0])
          first = int(weight.nonzero()[0, 0])
          drawn, low, high = (min(max(int((up <= w).sum()), first), last) for w in (want, want - close * float(up[-1]), want + close * float(up[-1])))
          may = low, high
      if keep:
        emitted.append(x)
        kept += 1
      else:
        emitted.append(drawn)
        break
    out.append((kept, emitted + [-1] * (row0[s + 1] - row0[s] - len(emitted)), near, may))
  return out


quantised = fp8_helpers.quantised
