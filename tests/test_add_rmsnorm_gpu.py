"""Residual sums with norms against the definition in 64 bits."""

import math

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import draft_helpers as ref

pytestmark = pytest.mark.gpu

CODE = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32, torch.float8_e4m3fn: _lib.E4M3}
BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def ptr(t):
  return None if t is None else t.data_ptr()


def call(x, residual, total, weight, offset, eps, out, scale, width=None, stream=None):
  stream = torch.cuda.current_stream().cuda_stream if stream is None else stream
  ld = lambda t: 0 if t is None else t.stride(0)
  _lib.check(_lib.load().mtx_add_rmsnorm(
      x.data_ptr(), CODE[x.dtype], ld(x), ptr(residual), 0 if residual is None else CODE[residual.dtype], ld(residual), ptr(total), ld(total), ptr(weight),
      0 if weight is None else CODE[weight.dtype], offset, eps, out.data_ptr(), CODE[out.dtype], ld(out), ptr(scale), x.shape[0], width or x.shape[1], stream))


def placed(t, shift, pitch):
  """t on the GPU, `shift` values behind 16 bytes, rows `pitch` values apart; around it a pattern."""
  rows, width = t.shape
  store = torch.full((rows * pitch + shift + 64,), 7.0, dtype=t.dtype, device="cuda")
  view = store[shift : shift + rows * pitch].as_strided((rows, width), (pitch, 1), shift)
  view.copy_(t)
  return store, view


def untouched(store, view, shift, pitch):
  """Whether the pattern around a view is still there."""
  mark = torch.ones_like(store, dtype=torch.bool)
  mark.as_strided(view.shape, view.stride(), shift).fill_(False)
  return bool((store[mark].float() == 7.0).all())


def check(x, residual, weight, offset, eps, total, out, scale):
  h, y = ref.normed(x.cpu(), None if residual is None else residual.cpu(), None if weight is None else weight.cpu(), offset, eps, None if residual is None else residual.dtype)
  if total is not None:
    assert torch.equal(total.cpu().double(), h)
  if out.dtype == FP8:
    ref.eight_bits(y, out.cpu().double(), scale.cpu().double())
  else:
    got = out.cpu().double()
    assert bool(((got - y).abs() <= (ref.EPS[out.dtype] + 2.0**-18) * y.abs() + 2.0**-130).all())


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 8), (5, 127), (9, 128), (4, 129), (17, 255), (8, 256), (3, 513), (7, 1000), (5, 1024), (6, 1025), (64, 1280), (3, 4095), (2, 4097), (3, 5376),
                                        (2, 16384), (2, 16391), (2, 32768)])
@pytest.mark.parametrize("types", [(BF16, BF16, FP8), (F32, F32, FP8), (BF16, F32, BF16), (F32, BF16, F32), (BF16, None, FP8), (F32, None, BF16)])
def test_shapes(rows, width, types):
  g = torch.Generator().manual_seed(rows * 100000 + width)
  tx, tr, to = types
  x = torch.randn(rows, width, generator=g).to(tx).cuda()
  residual = None if tr is None else (3 * torch.randn(rows, width, generator=g)).to(tr).cuda()
  weight = (1 + 0.3 * torch.randn(width, generator=g)).to(F32 if width % 2 else BF16).cuda()
  total = None if tr is None else torch.empty_like(residual)
  pitch = -(-width // 16) * 16
  out = torch.empty(rows, pitch, dtype=to, device="cuda")[:, :width]
  scale = torch.empty(rows, -(-width // 128), device="cuda") if to == FP8 else None
  call(x, residual, total, weight, 0.5, 1e-5, out, scale)
  check(x, residual, weight, 0.5, 1e-5, total, out, scale)


@pytest.mark.parametrize("width", [8200, 10001, 12289, 14336, 15353, 15361, 24577])
@pytest.mark.parametrize("types", [(BF16, BF16, FP8), (F32, F32, FP8), (BF16, F32, F32)])
def test_more_wide_rows_than_sms(width, types):
  g = torch.Generator("cuda").manual_seed(width)
  tx, tr, to = types
  rows = 150
  x = torch.randn(rows, width, generator=g, device="cuda").to(tx)
  residual = (3 * torch.randn(rows, width, generator=g, device="cuda")).to(tr)
  weight = 1 + 0.3 * torch.randn(width, generator=g, device="cuda")
  total = torch.empty_like(residual)
  out = torch.empty(rows, -(-width // 16) * 16, dtype=to, device="cuda")[:, :width]
  scale = torch.empty(rows, -(-width // 128), device="cuda") if to == FP8 else None
  call(x, residual, total, weight, 0.0, 1e-5, out, scale)
  check(x, residual, weight, 0.0, 1e-5, total, out, scale)


@pytest.mark.parametrize("first", [0, 1])
def test_largest_products_that_round_alike(first):
  """Of two neighbours whose products are the same number in 32 bits the larger one, by half a last bit, is a block's largest."""
  g = torch.Generator().manual_seed(3)
  x = torch.rand(512, 128, generator=g) - 0.5
  weight = torch.ones(128)
  x[:, 40 + first] = weight[40 + first] = 1 + 2.0**-12  # 1 + 2^-11 + 2^-24, an even number and half a last bit
  x[:, 41 - first] = 1 + 2.0**-11
  out = torch.empty(512, 128, dtype=FP8, device="cuda")
  scale = torch.empty(512, 1, device="cuda")
  call(x.cuda(), None, None, weight.cuda(), 0.0, 1e-5, out, scale)
  check(x.cuda(), None, weight.cuda(), 0.0, 1e-5, None, out, scale)
  # the mean is one of 32-bit sums of eight squares, of even and of odd places: 5 * 2^-24 off, more than what this looks for.  (A product and a sum in 64 bits, rounded once, are the fused step)
  squares = x.double().view(512, 16, 8)
  sums = torch.zeros(2, 512, 16)
  for i in range(8):
    sums[i % 2] = (squares[:, :, i] ** 2 + sums[i % 2].double()).float()
  mean = (sums[0] + sums[1]).double().sum(1) / 128
  want = (1 + 2.0**-12) ** 2 / (mean + float(torch.tensor(1e-5))).sqrt() / 448
  assert torch.equal(scale.cpu()[:, 0], want.float())


@pytest.mark.parametrize("shift", range(8))
@pytest.mark.parametrize("width", [5, 136, 777, 1031, 8200])
@pytest.mark.parametrize("types", [(BF16, BF16, BF16), (F32, F32, F32), (BF16, F32, BF16)])
def test_places(shift, width, types):
  """Rows at any place and pitch, each operand at another; nothing around the results changes."""
  g = torch.Generator().manual_seed(shift * 1000 + width)
  rows = 5
  tx, tr, to = types
  xs = torch.randn(rows, width, generator=g).to(tx)
  rs = torch.randn(rows, width, generator=g).to(tr)
  _, x = placed(xs, shift, width + shift)
  _, residual = placed(rs, (shift * 3) % 8, width + 1)
  total_store, total = placed(torch.zeros(rows, width, dtype=tr), (shift * 5) % 8, width + 3)
  out_store, out = placed(torch.zeros(rows, width, dtype=to), (shift + 2) % 8, width + (shift + 1) % 8)
  weight = torch.randn(width + 1, generator=g).cuda()[1:]
  call(x, residual, total, weight, 0.0, 1e-6, out, None)
  check(x, residual, weight, 0.0, 1e-6, total, out, None)
  assert untouched(total_store, total, (shift * 5) % 8, width + 3) and untouched(out_store, out, (shift + 2) % 8, width + (shift + 1) % 8)


def test_bytes_behind_a_row():
  rows, width = 6, 200
  x = torch.randn(rows, width, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF16)
  store = torch.full((rows, 256), 0x55, dtype=torch.uint8, device="cuda")
  scale = torch.empty(rows, 2, device="cuda")
  call(x, None, None, None, 0.0, 1e-5, store.view(FP8), scale, width=width)
  check(x, None, None, 0.0, 1e-5, None, store.view(FP8)[:, :width], scale)
  assert bool((store[:, width:] == 0x55).all())


@pytest.mark.parametrize("width", [1000, 1280, 5377])
def test_in_place(width):
  g = torch.Generator().manual_seed(width)
  x, residual = torch.randn(4, width, generator=g).to(BF16), torch.randn(4, width, generator=g).to(BF16)
  weight = torch.randn(width, generator=g).cuda()
  for where in ("sum is residual", "sum is x", "out is x", "both", "out is residual"):
    a, r = x.cuda(), residual.cuda()
    total = a if where == "sum is x" else None if where == "out is residual" else r
    out = a if where in ("out is x", "both") else r if where == "out is residual" else torch.empty_like(a)
    call(a, r, total, weight, 1.0, 1e-5, out, None)
    check(x, residual, weight, 1.0, 1e-5, total, out, None)


def test_sum_that_is_not_kept():
  x, residual = torch.randn(3, 300).to(BF16).cuda(), torch.randn(3, 300).cuda()
  before, out = residual.clone(), torch.empty(3, 300, device="cuda")
  call(x, residual, None, None, 0.0, 1e-5, out, None)
  check(x, residual, None, 0.0, 1e-5, None, out, None)
  assert torch.equal(before, residual)


@pytest.mark.parametrize("width", [100, 640, 1300])
def test_values_that_are_no_numbers(width):
  """A NaN makes its row NaN, an infinity its row 0 with a NaN in its place; rows of zeros stay zeros; the other rows are what they are without them."""
  x = torch.randn(6, width, generator=torch.Generator().manual_seed(width))
  x[1, 3], x[2, width - 1], x[3] = math.nan, math.inf, 0.0
  x[4] *= 2.0**-100
  clean = torch.where(x.isfinite(), x, 0.0)
  for to in (BF16, F32, FP8):
    outs = []
    for v in (x, clean):
      out = torch.zeros(6, -(-width // 128) * 128, dtype=to, device="cuda")
      scale = torch.zeros(6, -(-width // 128), device="cuda")
      call(v.cuda(), None, None, None, 0.0, 1e-5, out, scale if to == FP8 else None, width=width)
      outs.append((out[:, :width].float().cpu(), scale.cpu()))
    (got, scale), (want, clean_scale) = outs
    assert bool(got[1].isnan().all())
    assert bool(got[2, width - 1].isnan()) and (to == FP8 or bool((got[2, : width - 1] == 0).all()))
    assert bool((got[3] == 0).all())
    for r in (0, 3, 4, 5):
      assert torch.equal(got[r], want[r]) and torch.equal(scale[r], clean_scale[r])
    if to == FP8:
      assert bool(scale[1].isnan().all()) and bool(scale[2, -1].isnan()) and bool((scale[3] == torch.tensor(2.0**-96 / 448)).all())


def test_no_eps():
  x = torch.cat([torch.randn(1, 256), torch.zeros(1, 256)]).cuda()
  out, scale = torch.empty(2, 256, dtype=FP8, device="cuda"), torch.empty(2, 2, device="cuda")
  call(x, None, None, None, 0.0, 0.0, out, scale)
  check(x[:1], None, None, 0.0, 0.0, None, out[:1], scale[:1])
  assert bool(out[1].float().isnan().all())


def test_tiny_rows_with_a_tiny_eps():
  x = (2.0**-120 * torch.randn(2, 300, generator=torch.Generator().manual_seed(5))).cuda()
  x[:, 0] = 0
  out, scale = torch.empty(2, 304, dtype=FP8, device="cuda")[:, :300], torch.empty(2, 3, device="cuda")
  call(x, None, None, None, 0.0, 1e-38, out, scale)
  assert bool(out.float().isfinite().all()) and bool(scale.isfinite().all())


def test_rows_far_apart():
  """Rows whose values lie more than 2^31 apart."""
  pitch, width = (1 << 31) + 16, 640
  store = torch.empty(pitch + 1024, dtype=BF16, device="cuda")
  x = store.as_strided((2, width), (pitch, 1))
  x.copy_(torch.randn(2, width, generator=torch.Generator().manual_seed(2)))
  before = x.clone()
  out = torch.empty(2, width, device="cuda")
  call(x, before, x, None, 0.0, 1e-5, out, None)
  check(before, before, None, 0.0, 1e-5, x, out, None)


def test_streams_and_graphs():
  g = torch.Generator().manual_seed(9)
  x, residual = torch.randn(70, 1280, generator=g).to(BF16).cuda(), torch.randn(70, 1280, generator=g).to(BF16).cuda()
  keep = residual.clone()
  weight = torch.randn(1280, generator=g).cuda()
  out, scale = torch.empty(70, 1280, dtype=FP8, device="cuda"), torch.empty(70, 10, device="cuda")
  side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
  torch.cuda.synchronize()
  with torch.cuda.graph(graph, stream=side):
    call(x, residual, residual, weight, 0.0, 1e-5, out, scale)
  for _ in range(3):  # the residual stream grows with every replay
    before = residual.clone()
    graph.replay()
    torch.cuda.synchronize()
    check(x, before, weight, 0.0, 1e-5, residual, out, scale)
  assert not torch.equal(keep, residual)


def test_the_next_product_reads_it():
  """The 8-bit rows as mtx_linear_fp8 takes them: the same bytes as a quantisation of the fp32 result wherever no rounding lies between."""
  lib, g = _lib.load(), torch.Generator().manual_seed(4)
  rows, width, n = 33, 1280, 256
  x = torch.randn(rows, width, generator=g).cuda()
  out, scale = torch.empty(rows, width, dtype=FP8, device="cuda"), torch.empty(rows, 10, device="cuda")
  call(x, None, None, None, 0.0, 1e-5, out, scale)
  w = torch.randn(n, width, generator=g).cuda()
  wq, ws, y = torch.empty(n, width, dtype=torch.uint8, device="cuda"), torch.empty(n // 128, 10, device="cuda"), torch.empty(rows, n, device="cuda")
  stream = torch.cuda.current_stream().cuda_stream
  _lib.check(lib.mtx_quantize_fp8(w.data_ptr(), _lib.F32, width, n, width, 128, wq.data_ptr(), width, ws.data_ptr(), stream))
  _lib.check(lib.mtx_linear_fp8(out.data_ptr(), _lib.E4M3, width, scale.data_ptr(), wq.data_ptr(), width, ws.data_ptr(), y.data_ptr(), _lib.F32, n, rows, n, width, None, 0, stream))
  spread = lambda s, b, r: s.double().repeat_interleave(b, 0)[:r].repeat_interleave(128, 1)
  want = (out.double() * spread(scale, 1, rows)) @ (wq.view(FP8).double() * spread(ws, 128, n)).T
  size = (out.double().abs() * spread(scale, 1, rows)) @ (wq.view(FP8).double().abs() * spread(ws, 128, n)).T
  assert bool(((y.double() - want).abs() <= size * (132 * 2.0**-23 + 12 * 2.0**-24)).all())


@pytest.mark.parametrize("width", [100, 512, 1000, 1280, 5376, 8203, 20000])
@pytest.mark.parametrize("types", [(F32, None, BF16), (F32, F32, F32), (F32, F32, FP8), (BF16, BF16, BF16), (BF16, None, FP8), (BF16, BF16, FP8)])
@pytest.mark.parametrize("size", [62, 66, 90, 126, -49, -55, -70, -100])
def test_squares_beyond_32_bits(width, types, size):
  """Rows of values around 2^size, whose squares 32 bits do not hold, beside rows of ordinary ones and rows of both."""
  g = torch.Generator().manual_seed(width + size)
  tx, tr, to = types
  x = torch.randn(6, width, generator=g).clamp(-3.5, 3.5)
  residual = None if tr is None else torch.randn(6, width, generator=g).clamp(-3.5, 3.5)
  for r in (0, 2, 5):
    x[r] *= 2.0 ** (size - 2)
    if tr is not None:
      residual[r] *= 2.0 ** (size - 2)
  x[3, width // 2] = 2.0**size
  x, residual = x.to(tx), None if tr is None else residual.to(tr)
  weight = 1 + 0.3 * torch.randn(width, generator=g)
  eps = 0.0 if size < 0 else 1e-5
  pitch = -(-width // 16) * 16
  for where in ("apart", "in place") if to == BF16 else ("apart",):
    a, r = x.cuda(), None if residual is None else residual.cuda()
    total = None if r is None else r if where == "in place" else torch.empty_like(r)
    out = a if where == "in place" and tx == BF16 else torch.empty(6, pitch, dtype=to, device="cuda")[:, :width]
    scale = torch.empty(6, -(-width // 128), device="cuda") if to == FP8 else None
    call(a, r, total, weight.cuda(), 0.0, eps, out, scale)
    check(x, residual, weight, 0.0, eps, total, out, scale)
