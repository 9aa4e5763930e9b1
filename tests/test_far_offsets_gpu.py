"""Results and records whose elements lie more than 2^31 apart: the last rows of calls that large, against calls of their own."""

import pytest
import torch

from maxtext_indextts2_b200 import _lib

pytestmark = pytest.mark.gpu

ROWS, WIDE = 8200, 264192  # 2.17e9 values


@pytest.fixture(autouse=True)
def room():
  torch.cuda.empty_cache()
  if torch.cuda.mem_get_info()[0] < 60e9:
    pytest.skip("needs 60 GB of free device memory")
  yield
  torch.cuda.empty_cache()


def stream():
  return torch.cuda.current_stream().cuda_stream


def test_last_rows_of_a_quantisation():
  x = torch.randn(ROWS, WIDE, device="cuda", dtype=torch.bfloat16)
  lib = _lib.load()
  for block in (1, 128):
    q, s = torch.empty(ROWS, WIDE, dtype=torch.uint8, device="cuda"), torch.empty(-(-ROWS // block), WIDE // 128, device="cuda")
    _lib.check(lib.mtx_quantize_fp8(x.data_ptr(), _lib.BF16, WIDE, ROWS, WIDE, block, q.data_ptr(), WIDE, s.data_ptr(), stream()))
    last = ROWS % 128
    q1, s1 = torch.empty(last, WIDE, dtype=torch.uint8, device="cuda"), torch.empty(-(-last // block), WIDE // 128, device="cuda")
    tail = x[-last:].clone()
    _lib.check(lib.mtx_quantize_fp8(tail.data_ptr(), _lib.BF16, WIDE, last, WIDE, block, q1.data_ptr(), WIDE, s1.data_ptr(), stream()))
    assert torch.equal(q[-last:], q1) and torch.equal(s[-s1.shape[0] :], s1)


@pytest.mark.parametrize("k", [128, 300])
def test_last_rows_of_a_product(k):
  lib, g = _lib.load(), torch.Generator("cuda").manual_seed(1)
  w, pitch = torch.randn(WIDE, k, device="cuda", generator=g), -(-k // 16) * 16
  wq, ws = torch.empty(WIDE, pitch, dtype=torch.uint8, device="cuda"), torch.empty(WIDE // 128, -(-k // 128), device="cuda")
  _lib.check(lib.mtx_quantize_fp8(w.data_ptr(), _lib.F32, k, WIDE, k, 128, wq.data_ptr(), pitch, ws.data_ptr(), stream()))
  x = torch.randn(ROWS, k, device="cuda", generator=g).to(torch.bfloat16)

  def call(x, out):
    need = lib.mtx_linear_fp8_scratch_bytes(x.shape[0], k)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    _lib.check(lib.mtx_linear_fp8(x.data_ptr(), _lib.BF16, k, None, wq.data_ptr(), pitch, ws.data_ptr(), out.data_ptr(), _lib.F32, out.stride(0), x.shape[0], WIDE, k,
                                  scratch.data_ptr(), need, stream()))

  out, tail = torch.empty(ROWS, WIDE, device="cuda"), torch.empty(40, WIDE, device="cuda")
  call(x, out)
  call(x[-40:].clone(), tail)
  # (other tiles, the same order of the blocks: what the tensor cores' sums of 32 products may differ by)
  size = float((x[-40:].double().abs() @ w.double().abs().T).max())
  assert float((out[-40:] - tail).abs().max()) <= 2 * size * 132 * 2.0**-23
  assert float(out[-1].abs().max()) > 0


def test_last_rows_of_controlled_logits():
  lib, g = _lib.load(), torch.Generator("cuda").manual_seed(2)
  logits = torch.randn(ROWS, WIDE, device="cuda", generator=g)
  seen = torch.zeros(ROWS, WIDE, dtype=torch.int16, device="cuda")
  touched = torch.zeros(ROWS, WIDE // 256, dtype=torch.int32, device="cuda")
  token = torch.tensor([0, 7, WIDE - 1, WIDE - 1], dtype=torch.int32, device="cuda")
  slot = torch.full((4,), ROWS - 1, dtype=torch.int32, device="cuda")
  _lib.check(lib.mtx_note_tokens(seen.data_ptr(), WIDE, touched.data_ptr(), WIDE // 256, ROWS, WIDE, token.data_ptr(), slot.data_ptr(), 4, 0, stream()))
  assert seen[-1].nonzero()[:, 0].tolist() == [0, 7, WIDE - 1] and int(seen[-1, -1]) == 2 and int(seen[-2].count_nonzero()) == 0
  frequency = torch.full((ROWS,), 0.5, device="cuda")
  c = _lib.LogitControls(slots=ROWS, seen=seen.data_ptr(), ld_seen=WIDE, touched=touched.data_ptr(), ld_touched=WIDE // 256, frequency=frequency.data_ptr())
  want = logits[-1].clone()
  want[[0, 7]] -= 0.5
  want[-1] -= 1.0
  second = logits[-2].clone()
  _lib.check(lib.mtx_control_logits(logits.data_ptr(), WIDE, logits.data_ptr(), WIDE, ROWS, WIDE, c, stream()))
  assert torch.equal(logits[-1], want) and torch.equal(logits[-2], second)
