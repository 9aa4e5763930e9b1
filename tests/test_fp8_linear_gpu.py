"""8-bit values with a scale per block of 128 and products of them (csrc/fp8_linear.cuh) against their definition in 64 bits."""

import ctypes

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import fp8_helpers as ref

pytestmark = pytest.mark.gpu

CODES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
FILL = 0x55


def stream():
  return torch.cuda.current_stream().cuda_stream


def quantize(x, block_rows):
  rows, k = x.shape
  q = torch.full((rows, ref.pitch(k)), FILL, dtype=torch.uint8, device="cuda")
  scale = torch.full((-(-rows // block_rows), -(-k // 128)), -1.0, device="cuda")
  _lib.check(_lib.load().mtx_quantize_fp8(x.data_ptr(), CODES[x.dtype], x.stride(0), rows, k, block_rows, q.data_ptr(), q.stride(0), scale.data_ptr(), stream()))
  return q, scale


def values(q, k):
  return q[:, :k].contiguous().view(torch.float8_e4m3fn).double().cpu()


def linear(x, wq, ws, n, k, out_dtype=torch.bfloat16, x_scale=None, ldo=None, out=None):
  lib, rows = _lib.load(), x.shape[0]
  if out is None:
    out = torch.full((rows, ldo or n), 7.0, dtype=out_dtype, device="cuda")
  need = lib.mtx_linear_fp8_scratch_bytes(rows, k)
  scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
  code = _lib.E4M3 if x_scale is not None else CODES[x.dtype]
  _lib.check(lib.mtx_linear_fp8(x.data_ptr(), code, x.stride(0), None if x_scale is None else x_scale.data_ptr(), wq.data_ptr(), wq.stride(0), ws.data_ptr(), out.data_ptr(),
                                CODES[out.dtype], out.stride(0), rows, n, k, scratch.data_ptr(), need, stream()))
  return out


def inputs(rows, n, k, seed=0, dtype=torch.bfloat16):
  g = torch.Generator().manual_seed(seed + 1000003 * rows + 1009 * n + k)
  x = torch.randn(rows, k, generator=g) * torch.exp(torch.randn(rows, 1, generator=g)) * (1 + 20 * (torch.rand(k, generator=g) > 0.99))
  return x.to(dtype), torch.randn(n, k, generator=g) * k**-0.5


def expected(xq, xs, wq, ws, rows, n, k):
  """The product in 64 bits, and what a sum in fp32 may be off.  An MMA adds 32 products and the accumulator, each cut at 2^-23 of the largest at worst: 33 * 4 of
  those per block of 128; then a rounding of 2^-24 per block and two of the scales."""
  x, w = xq * ref.spread(xs, 1, rows, k), wq * ref.spread(ws, 128, n, k)
  return x @ w.T, (x.abs() @ w.abs().T) * (132 * 2.0**-23 + (-(-k // 128) + 2) * 2.0**-24)


def close(out, want, slack):
  """bfloat16 results are rounded once more (half a step: 2^-8 of the value, 2^-133 near zero)."""
  tol = slack + (want.abs() + slack) * (2.0**-8 if out.dtype == torch.bfloat16 else 2.0**-24) + 2.0**-133
  off = (out.double().cpu() - want).abs() - tol
  assert (off <= 0).all(), float(off.max())


# ---- quantisation -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 129), (5, 7), (127, 136), (128, 128), (129, 1280), (2, 1281), (300, 250), (33, 2560), (64, 1284)])
def test_values_and_scales(rows, k, block_rows, dtype):
  x, _ = inputs(rows, 1, k, dtype=dtype)
  q, scale = quantize(x.cuda(), block_rows)
  want_q, want_scale = ref.quantised(x, block_rows)
  assert torch.equal(scale.double().cpu(), want_scale)
  assert torch.equal(values(q, k), want_q)
  assert (q[:, k:] == FILL).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_strided_rows(block_rows, dtype):
  """Rows inside a wider matrix, from an odd column on, with a pitch of an odd number of values."""
  x, _ = inputs(37, 1, 701, dtype=dtype)
  part = x.cuda()[:, 3:603]
  q, scale = quantize(part, block_rows)
  want_q, want_scale = ref.quantised(x[:, 3:603], block_rows)
  assert torch.equal(values(q, 600), want_q) and torch.equal(scale.double().cpu(), want_scale)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_extreme_values(block_rows):
  """Zeros, the type's lowest and smallest values, infinities and NaN each keep to their block."""
  x = torch.randn(6, 512, generator=torch.Generator().manual_seed(5))
  x[0, :128] = 0
  x[1, 128:256] = 2.0**-130
  x[2, 256:384] = torch.finfo(torch.float32).max
  x[2, 300] = torch.finfo(torch.float32).min
  if block_rows == 1:
    x[3, 5] = float("inf")
    x[4, 200] = float("nan")
  else:
    x[3, 400] = float("nan")
  q, scale = quantize(x.cuda(), block_rows)
  want_q, want_scale = ref.quantised(x, block_rows)
  assert torch.equal(torch.nan_to_num(scale.double().cpu(), nan=-3.0), torch.nan_to_num(want_scale, nan=-3.0))
  assert torch.equal(torch.nan_to_num(values(q, 512), nan=-3.0), torch.nan_to_num(want_q, nan=-3.0))


def test_every_magnitude_rounds_as_defined():
  """All bfloat16 values of a binade range against a block maximum that is no multiple of 7 / 4: every border of the 8-bit type is met from both sides."""
  bits = torch.arange(0x3000, 0x43A0, dtype=torch.int32)
  x = (bits << 16).view(torch.float32)
  rows = -(-x.numel() // 127)
  full = torch.zeros(rows, 128)
  for r in range(rows):
    part = x[r * 127 : (r + 1) * 127]
    full[r, : part.numel()] = part * (1 if r % 2 else -1)
    full[r, 127] = 320.0 + r
  q, scale = quantize(full.cuda(), 1)
  want_q, want_scale = ref.quantised(full, 1)
  assert torch.equal(values(q, 128), want_q) and torch.equal(scale.double().cpu(), want_scale)


# ---- products ---------------------------------------------------------------------------------------------------------------------

SHAPES = [
    (1, 1, 1), (1, 16, 64), (1, 1792, 1280), (2, 129, 127), (7, 128, 128), (8, 300, 2048), (16, 1280, 5120), (17, 257, 640), (31, 130, 130), (33, 100, 1000),
    (64, 1280, 1281), (65, 512, 256), (100, 4000, 272), (127, 33, 3001), (128, 128, 128), (129, 128, 384), (200, 1000, 2560), (256, 256, 1024), (257, 255, 144),
    (333, 640, 1288), (500, 2051, 260), (700, 64, 4096), (1024, 384, 512), (1500, 700, 1100), (16, 60001, 100), (3, 70000, 384), (130, 20000, 300), (2049, 1300, 128),
]


@pytest.mark.parametrize("rows,n,k", SHAPES)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_product(rows, n, k, out_dtype):
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  out = linear(x.cuda(), wq, ws, n, k, out_dtype)
  xq, xs = ref.quantised(x, 1)
  close(out, *expected(xq, xs, values(wq, k), ws.double().cpu(), rows, n, k))


# Sums that several CTAs share (few rows and many), tiles of 128 and 256 columns in one wave and in several, pairs of CTAs in one wave and in two.
LARGER = [(20, 1300, 2600), (32, 300, 1300), (80, 150, 2100), (257, 1000, 3200), (500, 1500, 2048), (300, 10240, 1280), (1100, 8190, 1280), (1030, 2200, 2570), (2500, 2901, 1280)]


@pytest.mark.parametrize("rows,n,k", LARGER)
def test_larger_product(rows, n, k):
  """Both types of result, each at a pitch of whole 16 bytes and inside a wider matrix at an odd column whose other values stay."""
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  xq, xs = ref.quantised(x, 1)
  want = expected(xq, xs, values(wq, k), ws.double().cpu(), rows, n, k)
  for out_dtype in (torch.bfloat16, torch.float32):
    ldo = -(-n // 8) * 8
    out = linear(x.cuda(), wq, ws, n, k, out_dtype, ldo=ldo)
    close(out[:, :n], *want)
    assert (out[:, n:] == 7.0).all()
    whole = torch.full((rows + 3, ldo + 9), 7.0, dtype=out_dtype, device="cuda")
    linear(x.cuda(), wq, ws, n, k, out=whole[:rows, 3 : 3 + n])
    assert torch.equal(whole[:rows, 3 : 3 + n], out[:, :n])
    whole[:rows, 3 : 3 + n] = 7.0
    assert (whole == 7.0).all()


@pytest.mark.parametrize("rows,n,k", [(30, 300, 1300), (100, 300, 2100), (300, 10240, 1280), (1030, 2200, 2570)])
def test_rows_of_larger_products_do_not_disturb_each_other(rows, n, k):
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  plain = linear(x.cuda(), wq, ws, n, k, torch.float32)
  x[1], x[2, 100], x[3, k - 1], x[4] = float("nan"), float("inf"), float("nan"), 0.0
  out = linear(x.cuda(), wq, ws, n, k, torch.float32)
  assert out[1:4].isnan().all() and (out[4] == 0).all()
  keep = [0] + list(range(5, rows))
  assert torch.equal(out[keep], plain[keep])


@pytest.mark.parametrize("rows,n,k", [(1, 200, 200), (16, 128, 1280), (64, 640, 2000), (130, 300, 300), (513, 512, 1040)])
def test_forms_of_the_activations_agree(rows, n, k):
  """Values that the call quantises and values that were quantised before give the same bits; the bytes behind a row's end are not read as values."""
  x, w = inputs(rows, n, k, dtype=torch.float32)
  wq, ws = quantize(w.cuda(), 128)
  a = linear(x.cuda(), wq, ws, n, k, torch.float32)
  q, s = quantize(x.cuda(), 1)
  q[:, k:] = 0x7F  # NaN
  wq[:, k:] = 0x7F
  assert torch.equal(linear(q, wq, ws, n, k, torch.float32, x_scale=s), a)
  xb = x.to(torch.bfloat16)
  assert torch.equal(linear(xb.cuda(), wq, ws, n, k), linear(xb.float().cuda(), wq, ws, n, k))


@pytest.mark.parametrize("rows,n", [(1, 40), (64, 250), (129, 77), (300, 520)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_what_lies_around_the_result_stays(rows, n, out_dtype):
  """A result inside a wider matrix at an odd column; rows behind the last one and columns beside are as they were."""
  k = 384
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  whole = torch.full((rows + 3, n + 9), 7.0, dtype=out_dtype, device="cuda")
  linear(x.cuda(), wq, ws, n, k, out=whole[:rows, 3 : 3 + n])
  xq, xs = ref.quantised(x, 1)
  close(whole[:rows, 3 : 3 + n], *expected(xq, xs, values(wq, k), ws.double().cpu(), rows, n, k))
  whole[:rows, 3 : 3 + n] = 7.0
  assert (whole == 7.0).all()


@pytest.mark.parametrize("rows", [5, 100, 300])
def test_rows_do_not_disturb_each_other(rows):
  """A row's result does not depend on its neighbours: rows of NaN, infinities and zeros beside it leave it as it is."""
  n, k = 300, 640
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  plain = linear(x.cuda(), wq, ws, n, k, torch.float32)
  x[1], x[2, 100], x[3, 639], x[4] = float("nan"), float("inf"), float("nan"), 0.0
  out = linear(x.cuda(), wq, ws, n, k, torch.float32)
  assert out[1:4].isnan().all() and (out[4] == 0).all()
  keep = [0] + list(range(5, rows))
  assert torch.equal(out[keep], plain[keep])


@pytest.mark.parametrize("rows,n,k", [(16, 1280, 5120), (64, 33000, 256), (300, 1000, 1280)])
def test_same_bits_every_time(rows, n, k):
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  first = linear(x.cuda(), wq, ws, n, k)
  for _ in range(5):
    assert torch.equal(linear(x.cuda(), wq, ws, n, k), first)


def test_no_rows():
  x, w = inputs(1, 128, 128)
  wq, ws = quantize(w.cuda(), 128)
  assert linear(x.cuda()[:0], wq, ws, 128, 128).shape == (0, 128)
  q, s = quantize(x.cuda()[:0], 1)
  assert q.shape[0] == 0 and s.shape[0] == 0


@pytest.mark.parametrize("rows", [3, 64, 260])
def test_in_a_graph_and_on_another_stream(rows):
  """Two captured graphs with a scratch of their own, replayed on two streams at once and again with other inputs."""
  n, k = 1000, 1280
  x, w = inputs(rows, n, k)
  wq, ws = quantize(w.cuda(), 128)
  lib, sides = _lib.load(), []
  need = lib.mtx_linear_fp8_scratch_bytes(rows, k)
  for i in range(2):
    xi = (x * (i + 1)).cuda()
    out, scratch = torch.empty(rows, n, device="cuda"), torch.empty(need, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
      _lib.check(lib.mtx_linear_fp8(xi.data_ptr(), _lib.BF16, xi.stride(0), None, wq.data_ptr(), wq.stride(0), ws.data_ptr(), out.data_ptr(), _lib.F32, n, rows, n, k,
                                    scratch.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    sides.append((xi, out, scratch, s, g))
  for again in range(2):
    for xi, out, scratch, s, g in sides:
      s.wait_stream(torch.cuda.current_stream())
      with torch.cuda.stream(s):
        g.replay()
    torch.cuda.synchronize()
    for xi, out, scratch, s, g in sides:
      assert torch.equal(out, linear(xi, wq, ws, n, k, torch.float32))
      xi.mul_(-0.5)
    torch.cuda.synchronize()


def test_calls_side_by_side():
  """Products of every kernel on three streams at once, each with a scratch of its own, give what they give alone."""
  shapes = [(1, 1792, 1280), (16, 2560, 5120), (30, 40000, 384), (64, 1280, 5120), (100, 640, 2048), (300, 1000, 1280), (700, 3000, 900), (2000, 2560, 640)]
  cases = []
  for rows, n, k in shapes:
    x, w = inputs(rows, n, k)
    wq, ws = quantize(w.cuda(), 128)
    cases.append((x.cuda(), wq, ws, n, k, torch.float32))
  alone = [linear(*c) for c in cases]
  torch.cuda.synchronize()
  streams, got = [torch.cuda.Stream() for _ in range(3)], []
  for i in range(60):
    which = (i * 5 + i // 7) % len(cases)
    with torch.cuda.stream(streams[i % 3]):
      got.append((which, linear(*cases[which])))
  torch.cuda.synchronize()
  for which, out in got:
    assert torch.equal(out, alone[which])


def test_refuses_memory_of_the_host():
  lib = _lib.load()
  x, q, s = torch.zeros(4, 128), torch.zeros(4, 128, dtype=torch.uint8, device="cuda"), torch.zeros(4, 1, device="cuda")
  assert lib.mtx_quantize_fp8(x.data_ptr(), _lib.F32, 128, 4, 128, 1, q.data_ptr(), 128, s.data_ptr(), stream()) == _lib.MTX_ERR_ARG
  assert "not device memory" in _lib.last_error()
  x = x.pin_memory()  # (the tensor copies of a product want device memory)
  assert lib.mtx_quantize_fp8(x.data_ptr(), _lib.F32, 128, 4, 128, 1, q.data_ptr(), 128, s.data_ptr(), stream()) == _lib.MTX_ERR_ARG


def test_no_wait_ran_out():
  count = ctypes.c_uint32(7)
  _lib.check(_lib.load().mtx_linear_fp8_stalls(ctypes.byref(count)))
  assert count.value == 0


def test_stalls_are_counted_behind_all_streams():
  """The count is read once every product in flight is done, on a stream of the caller's own too; products of every kernel waited for nothing in vain."""
  side, lib, count = torch.cuda.Stream(), _lib.load(), ctypes.c_uint32(7)
  for rows, n, k, times in [(1, 1792, 1280, 50), (30, 40000, 384, 50), (64, 1280, 5120, 50), (100, 640, 2048, 50), (300, 10240, 1280, 50), (2048, 10240, 5120, 40)]:
    x, w = torch.randn(rows, k, device="cuda").to(torch.bfloat16), torch.randn(n, k, device="cuda")
    wq, ws = quantize(w, 128)
    need = lib.mtx_linear_fp8_scratch_bytes(rows, k)
    out, scratch = torch.empty(rows, n, device="cuda"), torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
      for _ in range(times):
        _lib.check(lib.mtx_linear_fp8(x.data_ptr(), _lib.BF16, k, None, wq.data_ptr(), wq.stride(0), ws.data_ptr(), out.data_ptr(), _lib.F32, n, rows, n, k, scratch.data_ptr(), need,
                                      stream()))
      done = side.record_event()
    _lib.check(lib.mtx_linear_fp8_stalls(ctypes.byref(count)))
    assert done.query() and count.value == 0
