"""The definitions of the 8-bit values and of the logit controls in 64 bits, on the CPU, for the tests."""

import torch

BLOCK = 128


def e4m3(v):
  """Nearest value of float8_e4m3fn (ties to even, at most 448 in size) of float64 values; NaN stays NaN."""
  size = v.abs()
  _, e = torch.frexp(torch.where(torch.isfinite(size), size, torch.ones_like(size)))
  step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
  return torch.where(torch.isnan(v), v, torch.sign(v) * torch.clamp(torch.round(size / step) * step, max=448.0))


def quantised(x, block_rows):
  """(values, scales) of x [rows, k], in float64; the two fractions and the scaled value are fp32 numbers."""
  rows, k = x.shape
  x = x.double()
  q = torch.empty_like(x)
  scales = torch.empty(-(-rows // block_rows), -(-k // BLOCK), dtype=torch.float64)
  for i in range(scales.shape[0]):
    for b in range(scales.shape[1]):
      at = (slice(i * block_rows, (i + 1) * block_rows), slice(b * BLOCK, (b + 1) * BLOCK))
      part = x[at].abs()
      largest = torch.tensor(float("nan"), dtype=torch.float64) if part.isnan().any() else part.max().clamp(min=2.0**-96)
      scales[i, b] = (largest / 448).float().double()
      q[at] = e4m3((x[at] * (448 / largest).float().double()).float().double())
  return q, scales


def spread(scales, block_rows, rows, k):
  return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :k]


def pitch(k):
  return -(-k // 16) * 16


def padded(q, fill=0x55):
  """float64 e4m3 values [rows, k] as 8-bit rows at a pitch of whole 16 bytes, the bytes between them `fill`."""
  rows, k = q.shape
  t = torch.full((rows, pitch(k)), fill, dtype=torch.uint8)
  t[:, :k] = q.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)
  return t


def controlled(logits, word, repetition, presence, frequency, bias, allowed):
  """One row in float64: word [vocab] ints, bias {token: value}, allowed [vocab] bools or None."""
  l = logits.double().clone()
  count = (word & 0x7FFF).double()
  l = torch.where(word != 0, torch.where(l > 0, l / repetition, l * repetition), l)
  l = torch.where(word != 0, l - frequency * count - presence * (count > 0), l)
  for t, v in bias.items():
    l[t] += v
  return l if allowed is None else torch.where(allowed, l, float("-inf"))
