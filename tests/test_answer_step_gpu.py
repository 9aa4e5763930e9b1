"""The answering end of a decode step as a server runs it: hidden states, 8-bit product over the vocabulary, controls, sampler, record of the drawn tokens."""

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import fp8_helpers as ref

pytestmark = pytest.mark.gpu


class Server:
  """Requests in slots of a record; a step is one captured graph over buffers that stay."""

  def __init__(self, rows, k, vocab, seed=3):
    g = torch.Generator().manual_seed(seed)
    self.lib = _lib.load()
    self.rows, self.k, self.vocab, self.slots = rows, k, vocab, rows + 3
    lib, w = self.lib, torch.randn(vocab, k, generator=g) * k**-0.5
    self.wq = torch.empty(vocab, ref.pitch(k), dtype=torch.uint8, device="cuda")
    self.ws = torch.empty(-(-vocab // 128), -(-k // 128), device="cuda")
    w = w.to(torch.bfloat16).cuda()
    _lib.check(lib.mtx_quantize_fp8(w.data_ptr(), _lib.BF16, k, vocab, k, 128, self.wq.data_ptr(), self.wq.stride(0), self.ws.data_ptr(), self.stream()))
    self.hidden = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    self.logits = torch.empty(rows, vocab, device="cuda")
    self.scratch = torch.empty(lib.mtx_linear_fp8_scratch_bytes(rows, k), dtype=torch.uint8, device="cuda")
    self.sample_scratch = torch.empty(5 * rows, device="cuda")
    self.rng = torch.tensor([1, 2, 3, 0], dtype=torch.int32, device="cuda")
    self.token, self.log_prob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    self.slot = torch.randperm(self.slots, generator=g)[:rows].int()
    self.slot_dev = self.slot.cuda()
    self.seen = torch.zeros(self.slots, -(-vocab // 8) * 8, dtype=torch.int16, device="cuda")
    self.touched = torch.zeros(self.slots, -(-vocab // 256), dtype=torch.int32, device="cuda")
    self.penalties = 1 + 4 * torch.rand(self.slots, generator=g), torch.rand(self.slots, generator=g), torch.rand(self.slots, generator=g)
    self.keep = [t.cuda() for t in self.penalties]
    self.allowed = torch.stack([torch.arange(vocab) >= vocab // 2, torch.rand(vocab, generator=g) < 0.05])
    bits = torch.zeros(2, -(-vocab // 32) * 32, dtype=torch.int64)
    bits[:, :vocab] = self.allowed
    self.mask = (bits.view(2, -1, 32) << torch.arange(32)).sum(-1).to(torch.int32).cuda()
    self.mask_row = (torch.arange(rows) % 3 - 1).int()  # every third row is free
    self.mask_row_dev = self.mask_row.cuda()
    self.bias = [{int(t): float(torch.tensor(v)) for t, v in zip(torch.randperm(vocab, generator=g)[:r].tolist(), torch.randn(r, generator=g).tolist())} for r in range(rows)]
    pairs = [sorted(b.items()) for b in self.bias]
    self.bias_off = torch.tensor([sum(len(b) for b in pairs[:r]) for r in range(rows + 1)], dtype=torch.int32).cuda()
    self.bias_token = torch.tensor([t for b in pairs for t, _ in b] + [0], dtype=torch.int32).cuda()
    self.bias_value = torch.tensor([v for b in pairs for _, v in b] + [0.0]).cuda()
    self.controls = _lib.LogitControls(
        slots=self.slots, slot=self.slot_dev.data_ptr(), seen=self.seen.data_ptr(), ld_seen=self.seen.stride(0), touched=self.touched.data_ptr(), ld_touched=self.touched.stride(0),
        repetition=self.keep[0].data_ptr(), presence=self.keep[1].data_ptr(), frequency=self.keep[2].data_ptr(), bias_off=self.bias_off.data_ptr(),
        bias_token=self.bias_token.data_ptr(), bias_value=self.bias_value.data_ptr(), allowed_rows=2, allowed_row=self.mask_row_dev.data_ptr(), allowed=self.mask.data_ptr(),
        ld_allowed=self.mask.stride(0))

  def stream(self):
    return torch.cuda.current_stream().cuda_stream

  def note(self, token, slot, prompt):
    _lib.check(self.lib.mtx_note_tokens(self.seen.data_ptr(), self.seen.stride(0), self.touched.data_ptr(), self.touched.stride(0), self.slots, self.vocab, token.data_ptr(),
                                        slot.data_ptr(), len(token), int(prompt), self.stream()))

  def step(self):
    lib = self.lib
    _lib.check(lib.mtx_linear_fp8(self.hidden.data_ptr(), _lib.BF16, self.k, None, self.wq.data_ptr(), self.wq.stride(0), self.ws.data_ptr(), self.logits.data_ptr(), _lib.F32,
                                  self.vocab, self.rows, self.vocab, self.k, self.scratch.data_ptr(), self.scratch.numel(), self.stream()))
    _lib.check(lib.mtx_control_logits(self.logits.data_ptr(), self.vocab, self.logits.data_ptr(), self.vocab, self.rows, self.vocab, self.controls, self.stream()))
    _lib.check(lib.mtx_sample_rows(self.logits.data_ptr(), self.rows, self.vocab, self.vocab, _lib.SAMPLING["greedy"], 0, 0.0, 1.0, self.rng.data_ptr(), 0,
                                   self.sample_scratch.data_ptr(), self.token.data_ptr(), self.log_prob.data_ptr(), self.stream()))
    self.note(self.token, self.slot_dev, False)


@pytest.mark.parametrize("rows,k,vocab", [(1, 128, 777), (7, 640, 3001), (70, 200, 1024), (130, 384, 2050)])
@pytest.mark.parametrize("captured", [False, True])
def test_greedy_answers(rows, k, vocab, captured):
  s = Server(rows, k, vocab)
  g = torch.Generator().manual_seed(rows)
  prompt = torch.randint(0, vocab, (rows * 20,), generator=g).int()
  s.note(prompt.cuda(), s.slot_dev.repeat_interleave(20), True)
  words = torch.zeros(s.seen.shape, dtype=torch.int64)
  for t, slot in zip(prompt.tolist(), s.slot.repeat_interleave(20).tolist()):
    words[slot, t] |= 0x8000
  if captured:
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    s.hidden.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
      s.step()
  wq = s.wq[:, :k].contiguous().view(torch.float8_e4m3fn).double().cpu()
  w = wq * ref.spread(s.ws.double().cpu(), 128, vocab, k)
  hidden = torch.randn(rows, k, generator=g).to(torch.bfloat16)
  for step in range(6):  # the same hidden states: only the penalties move the answers on
    s.hidden.copy_(hidden)
    graph.replay() if captured else s.step()
    token = s.token.cpu().tolist()
    q, scale = ref.quantised(hidden, 1)
    x = q * ref.spread(scale, 1, rows, k)
    logits, size = x @ w.T, (x.abs() @ w.abs().T).max()
    slack = float(size) * (132 * 2.0**-23 + (-(-k // 128) + 2) * 2.0**-24) * 5  # of the product, grown by a penalty of at most 5
    for r in range(rows):
      slot, m = int(s.slot[r]), int(s.mask_row[r])
      pen = [float(p[slot]) for p in s.penalties]
      want = ref.controlled(logits[r], words[slot, :vocab], *pen, s.bias[r], s.allowed[m] if m >= 0 else None)
      count = 6 * pen[2] + pen[1] + 4 * float(logits[r].abs().max())  # what a rounding is measured by
      assert m < 0 or bool(s.allowed[m][token[r]])
      assert float(want[token[r]]) >= float(want.max()) - 2 * (slack + 5 * 2.0**-24 * (count + 5))
      words[slot, token[r]] = words[slot, token[r]] & 0x8000 | (words[slot, token[r]] & 0x7FFF) + 1
    assert torch.equal(s.seen.cpu().long() & 0xFFFF, words)
  assert len(set(token)) > 0 and int((words & 0x7FFF).sum()) == 6 * rows


def test_weights_of_the_call_in_front():
  """Weights that one call writes are the ones that the next call reads, whether it quantises its activations or not."""
  lib, n, k = _lib.load(), 4000, 2048
  stream = torch.cuda.current_stream().cuda_stream
  wq, ws = torch.empty(n, k, dtype=torch.uint8, device="cuda"), torch.empty(-(-n // 128), k // 128, device="cuda")
  for rows in (1, 64, 300):
    x = torch.randn(rows, k, device="cuda", generator=torch.Generator("cuda").manual_seed(rows)).to(torch.bfloat16)
    need = lib.mtx_linear_fp8_scratch_bytes(rows, k)
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    xq, xs = torch.empty(rows, k, dtype=torch.uint8, device="cuda"), torch.empty(rows, k // 128, device="cuda")
    _lib.check(lib.mtx_quantize_fp8(x.data_ptr(), _lib.BF16, k, rows, k, 1, xq.data_ptr(), k, xs.data_ptr(), stream))

    def call(out, quantised):
      a, s, code = (xq, xs.data_ptr(), _lib.E4M3) if quantised else (x, None, _lib.BF16)
      _lib.check(lib.mtx_linear_fp8(a.data_ptr(), code, k, s, wq.data_ptr(), k, ws.data_ptr(), out.data_ptr(), _lib.F32, n, rows, n, k, scratch.data_ptr(), need, stream))

    weights = [torch.randn(n, k, device="cuda", generator=torch.Generator("cuda").manual_seed(i)) for i in range(4)]
    outs = [torch.empty(rows, n, device="cuda") for _ in range(16)]
    for i, out in enumerate(outs):
      w = weights[i % 4]
      _lib.check(lib.mtx_quantize_fp8(w.data_ptr(), _lib.F32, k, n, k, 128, wq.data_ptr(), k, ws.data_ptr(), stream))
      call(out, i % 2 == 0 if i < 8 else i % 2 == 1)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
      w = weights[i % 4]
      _lib.check(lib.mtx_quantize_fp8(w.data_ptr(), _lib.F32, k, n, k, 128, wq.data_ptr(), k, ws.data_ptr(), stream))
      torch.cuda.synchronize()
      again = torch.empty(rows, n, device="cuda")
      call(again, True)
      torch.cuda.synchronize()
      assert torch.equal(out, again)
