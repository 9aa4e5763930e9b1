"""Penalties, biases and masks on a batch's logits, and the record of seen tokens (csrc/logit_controls.cuh), against their definition in 64 bits."""

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import fp8_helpers as ref

pytestmark = pytest.mark.gpu


def stream():
  return torch.cuda.current_stream().cuda_stream


def record(slots, vocab):
  return torch.zeros(slots, -(-vocab // 8) * 8, dtype=torch.int16, device="cuda"), torch.zeros(slots, -(-vocab // 256), dtype=torch.int32, device="cuda")


def note(seen, touched, vocab, token, slot, prompt):
  token = torch.as_tensor(token, dtype=torch.int32).cuda()
  slot = None if slot is None else torch.as_tensor(slot, dtype=torch.int32).cuda()
  _lib.check(_lib.load().mtx_note_tokens(seen.data_ptr(), seen.stride(0), None if touched is None else touched.data_ptr(), 0 if touched is None else touched.stride(0), seen.shape[0],
                                         vocab, token.data_ptr(), None if slot is None else slot.data_ptr(), len(token), int(prompt), stream()))


def noted(words, vocab, token, slot, prompt):
  """The record's definition, token by token on the CPU."""
  for t, s in zip(token, slot):
    if 0 <= t < vocab and 0 <= s < words.shape[0]:
      w = int(words[s, t]) & 0xFFFF
      words[s, t] = w | 0x8000 if prompt else w & 0x8000 | min((w & 0x7FFF) + 1, 0x7FFF)


def touched_of(words):
  slots, ld = words.shape
  out = torch.zeros(slots, -(-ld // 256), dtype=torch.int64)
  for s, t in (words != 0).nonzero().tolist():
    out[s, t // 256] |= 1 << (t // 8 % 32)
  return out


class Batch:
  """A batch's logits and controls; the arrays live as long as the object."""

  def __init__(self, rows, vocab, *, history=40, biases=5, masks=3, seed=0, ld=None, offset=0, with_touched=True):
    g = torch.Generator().manual_seed(seed + 131 * rows + vocab)
    self.rows, self.vocab = rows, vocab
    ld = ld or vocab
    self.wide = torch.randn(rows * ld + offset + 8, generator=g).mul_(4).cuda()
    self.logits = self.wide[offset : offset + rows * ld].view(rows, ld)[:, :vocab]
    slots = rows + 2
    self.slot = torch.randperm(slots, generator=g)[:rows].int()
    if rows > 3:
      self.slot[3] = -1  # no penalties
    self.seen, self.touched = record(slots, vocab)
    if history:
      token = torch.randint(0, vocab, (slots * history,), generator=g)
      token[::7] = token[0]
      slot = torch.arange(slots).repeat_interleave(history)
      for prompt in (True, False):
        note(self.seen, self.touched, vocab, token[prompt::2], slot[prompt::2], prompt)
    if not with_touched:
      self.touched = None
    self.repetition = 1 + torch.rand(slots, generator=g) * 5
    self.presence, self.frequency = torch.rand(slots, generator=g), torch.rand(slots, generator=g)
    self.repetition[0], self.presence[0], self.frequency[0] = 1, 0, 0
    self.bias = [{int(t): float(v) for t, v in zip(torch.randperm(vocab, generator=g)[:biases].tolist(), 5 * torch.randn(biases, generator=g))} for _ in range(rows)]
    if rows > 1:
      self.bias[1] = {}
    self.allowed = None
    if masks:
      self.allowed = torch.rand(masks, vocab, generator=g) < 0.3
      self.allowed[0] = torch.arange(vocab) >= vocab // 2
      self.allowed[-1] = False
      self.allowed_row = torch.randint(-1, masks, (rows,), generator=g).int()
      self.allowed_row[rows // 2] = masks - 1
      words = -(-vocab // 32)
      full = torch.zeros(masks, words * 32, dtype=torch.int64)
      full[:, :vocab] = self.allowed
      self.mask = (full.view(masks, words, 32) << torch.arange(32)).sum(-1).to(torch.int32).cuda()
    self.keep = dict(slot=self.slot.cuda(), repetition=self.repetition.cuda(), presence=self.presence.cuda(), frequency=self.frequency.cuda())
    pairs = [sorted(b.items()) for b in self.bias]
    self.keep["bias_off"] = torch.tensor([0] + torch.tensor([len(b) for b in pairs]).cumsum(0).tolist(), dtype=torch.int32).cuda()
    self.keep["bias_token"] = torch.tensor([t for b in pairs for t, _ in b] + [0], dtype=torch.int32).cuda()
    self.keep["bias_value"] = torch.tensor([v for b in pairs for _, v in b] + [0.0]).cuda()
    if masks:
      self.keep["allowed_row"] = self.allowed_row.cuda()

  def controls(self, **other):
    k = {n: t.data_ptr() for n, t in self.keep.items()}
    k |= dict(slots=self.seen.shape[0], seen=self.seen.data_ptr(), ld_seen=self.seen.stride(0))
    if self.touched is not None:
      k |= dict(touched=self.touched.data_ptr(), ld_touched=self.touched.stride(0))
    if self.allowed is not None:
      k |= dict(allowed=self.mask.data_ptr(), allowed_rows=self.mask.shape[0], ld_allowed=self.mask.stride(0))
    return _lib.LogitControls(**{**k, **other})

  def run(self, out, **other):
    _lib.check(_lib.load().mtx_control_logits(self.logits.data_ptr(), self.logits.stride(0), out.data_ptr(), out.stride(0), self.rows, self.vocab, self.controls(**other), stream()))

  def want(self):
    logits, seen = self.logits.cpu(), self.seen.cpu().int() & 0xFFFF
    rows = []
    for r in range(self.rows):
      s = int(self.slot[r])
      a = int(self.allowed_row[r]) if self.allowed is not None else -1
      word = seen[s, : self.vocab] if s >= 0 else torch.zeros(self.vocab, dtype=torch.int32)
      rep, pre, fre = (float(v[s]) if s >= 0 else d for v, d in ((self.repetition, 1.0), (self.presence, 0.0), (self.frequency, 0.0)))
      bias = {t: float(torch.tensor(v)) for t, v in self.bias[r].items()}
      rows.append(ref.controlled(logits[r], word, rep, pre, fre, bias, self.allowed[a] if a >= 0 else None))
    return torch.stack(rows)


def close(got, want, batch):
  """Five fp32 roundings, none of a number larger than the logit times the penalty, the two penalties and the bias together."""
  got = got.double().cpu()
  assert torch.equal(got.isinf(), want.isinf()) and not got.isnan().any()
  count = int((batch.seen.cpu().int() & 0x7FFF).max())
  largest = float(batch.logits.abs().max()) * float(batch.repetition.max()) + count * float(batch.frequency.max()) + 1 + max([abs(v) for b in batch.bias for v in b.values()] + [0])
  finite = ~want.isinf()
  assert ((got - want)[finite].abs() <= 5 * 2.0**-24 * largest).all()


SIZES = [(1, 1), (1, 31), (2, 32), (3, 255), (5, 256), (1, 257), (4, 1000), (7, 8191), (2, 8192), (3, 8193), (64, 5001), (300, 700), (2, 33000)]


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_controls(rows, vocab, in_place):
  b = Batch(rows, vocab, biases=min(5, vocab))
  want = b.want()
  out = b.logits if in_place else torch.full((rows, vocab), 9.0, device="cuda")
  b.run(out)
  close(out, want, Batch(rows, vocab, biases=min(5, vocab)))


@pytest.mark.parametrize("ld,offset", [(1003, 0), (1004, 0), (1000, 1), (1000, 4), (1001, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pitch_and_alignment(ld, offset, in_place):
  """Rows inside a wider matrix, aligned or not; what lies beside them stays."""
  b = Batch(6, 999, ld=ld, offset=offset)
  want, before = b.want(), b.wide.clone()
  out = b.logits if in_place else torch.full((6, 1010), 9.0, device="cuda")[:, 3:1002] if offset % 2 else torch.full((6, 1012), 9.0, device="cuda")[:, :999]
  b.run(out)
  close(out, want, Batch(6, 999, ld=ld, offset=offset))
  if in_place:
    b.logits.copy_(before[offset : offset + 6 * ld].view(6, ld)[:, :999])
  assert torch.equal(b.wide, before)


def test_parts_that_are_left_out():
  """Without the bits per eight tokens the record is read whole; without penalties, biases or masks the rest applies; with nothing the logits are copied."""
  b = Batch(9, 3001)
  full, other = torch.empty(9, 3001, device="cuda"), torch.empty(9, 3001, device="cuda")
  b.run(full)
  b.run(other, touched=None)
  assert torch.equal(full, other)
  nothing = _lib.LogitControls()
  _lib.check(_lib.load().mtx_control_logits(b.logits.data_ptr(), 3001, other.data_ptr(), 3001, 9, 3001, nothing, stream()))
  assert torch.equal(other, b.logits)
  b.run(other, seen=None, repetition=None, presence=None, frequency=None, bias_off=None, bias_token=None, bias_value=None)
  want = torch.where(torch.stack([b.allowed[a] if a >= 0 else torch.ones(3001, dtype=torch.bool) for a in b.allowed_row.tolist()]).cuda(), b.logits, float("-inf"))
  assert torch.equal(other, want)
  b.run(other, allowed=None, bias_off=None, bias_token=None, bias_value=None, presence=None, frequency=None)
  seen = torch.stack([b.seen[s] if s >= 0 else torch.zeros_like(b.seen[0]) for s in b.slot.tolist()])[:, :3001] != 0
  rep = torch.tensor([float(b.repetition[s]) if s >= 0 else 1.0 for s in b.slot.tolist()]).cuda()[:, None]
  assert torch.equal(other, torch.where(seen, torch.where(b.logits > 0, b.logits / rep, b.logits * rep), b.logits))


@pytest.mark.parametrize("vec", [True, False])
def test_values_that_are_no_numbers(vec):
  """Infinities and NaN in masked places become -infinity; in others they go through the same arithmetic; the type's lowest value stays finite."""
  vocab = 1024 if vec else 1023
  b = Batch(4, vocab, history=0, biases=0)
  b.allowed_row[:] = torch.tensor([0, 0, -1, -1], dtype=torch.int32)
  b.keep["allowed_row"] = b.allowed_row.cuda()
  half = vocab // 2
  b.logits[0, 3], b.logits[0, 4], b.logits[1, 5] = float("nan"), float("inf"), torch.finfo(torch.float32).min
  b.logits[0, half + 9], b.logits[2, 7], b.logits[2, 8], b.logits[3, 9] = float("nan"), float("-inf"), float("inf"), torch.finfo(torch.float32).min
  out = torch.empty(4, vocab, device="cuda")
  b.run(out)
  assert (out[:2, :half] == float("-inf")).all()
  assert out[0, half + 9].isnan() and out[2, 7] == float("-inf") and out[2, 8] == float("inf") and out[3, 9] == torch.finfo(torch.float32).min
  assert not out[1:].isnan().any() and int(out[0].isnan().sum()) == 1


@pytest.mark.parametrize("in_place", [False, True])
def test_lists_of_biases(in_place):
  """Lists of none, one and very many entries, tokens outside the vocabulary, one token several times (its first entry counts), and biases of masked tokens."""
  vocab = 40000
  b = Batch(4, vocab, history=0, biases=0, masks=1)
  b.allowed[0] = torch.arange(vocab) % 3 != 0
  full = torch.zeros(1, vocab, dtype=torch.int64)
  full[:] = b.allowed
  b.mask = (full.view(1, -1, 32) << torch.arange(32)).sum(-1).to(torch.int32).cuda()
  b.allowed_row[:] = torch.tensor([0, -1, 0, -1], dtype=torch.int32)
  b.keep["allowed_row"] = b.allowed_row.cuda()
  lists = [list(range(vocab)), [], [-5, -1, 0, 1, 1, 1, 8191, 8191, 8192, vocab - 1, vocab, vocab + 7], [17] * 100 + [18]]
  b.keep["bias_off"] = torch.tensor([0, vocab, vocab, vocab + 12, vocab + 113], dtype=torch.int32).cuda()
  b.keep["bias_token"] = torch.tensor(sum(lists, []), dtype=torch.int32).cuda()
  value = torch.randn(vocab + 113, generator=torch.Generator().manual_seed(1))
  b.keep["bias_value"] = value.cuda()
  add, at = torch.zeros(4, vocab), 0
  for r, tokens in enumerate(lists):
    for i, t in enumerate(tokens):
      if 0 <= t < vocab and (i == 0 or tokens[i - 1] != t):
        add[r, t] = value[at + i]
    at += len(tokens)
  want = b.logits.cpu() + add
  want[::2][:, ~b.allowed[0]] = float("-inf")
  out = b.logits if in_place else torch.empty(4, vocab, device="cuda")
  b.run(out)
  assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("slots,vocab,n", [(1, 1, 5), (3, 9, 100), (4, 300, 1), (5, 5001, 3000), (64, 70, 64), (2, 257, 513)])
@pytest.mark.parametrize("prompt", [True, False])
def test_noted_tokens(slots, vocab, n, prompt):
  g = torch.Generator().manual_seed(n)
  seen, touched = record(slots, vocab)
  words = torch.zeros(seen.shape, dtype=torch.int32)
  for kind in (prompt, not prompt, prompt):
    token, slot = torch.randint(-2, vocab + 2, (n,), generator=g).tolist(), torch.randint(-1, slots + 1, (n,), generator=g).tolist()
    note(seen, touched, vocab, token, slot, kind)
    noted(words, vocab, token, slot, kind)
  assert torch.equal(seen.cpu().int() & 0xFFFF, words)
  assert torch.equal(touched.cpu().long() & 0xFFFFFFFF, touched_of(words))


def test_counts_stop_at_their_largest():
  """One token 70,000 times in two slots that share a word with another token's: the count stays at 32767, the prompt's bit and the neighbour are as they were."""
  seen, touched = record(2, 10)
  note(seen, touched, 10, [4, 5], [0, 1], True)
  note(seen, touched, 10, [5] * 3, [0] * 3, False)
  note(seen, touched, 10, [4] * 70000, [0, 1] * 35000, False)
  w = seen.cpu().int() & 0xFFFF
  assert int(w[0, 4]) == 0xFFFF and int(w[1, 4]) == 0x7FFF and int(w[0, 5]) == 3 and int(w[1, 5]) == 0x8000
  assert touched.cpu().tolist() == [[1], [1]]


def test_tokens_in_pinned_memory_and_refused_memory():
  """Lists that a server fills on the host may be pinned memory; memory that the device cannot read is refused."""
  lib, (seen, touched) = _lib.load(), record(2, 100)
  token = torch.tensor([3, 99], dtype=torch.int32).pin_memory()
  call = lambda t: lib.mtx_note_tokens(seen.data_ptr(), seen.stride(0), touched.data_ptr(), touched.stride(0), 2, 100, t.data_ptr(), None, 2, 0, stream())  # noqa: E731
  assert call(token) == _lib.MTX_OK
  assert seen.cpu().nonzero().tolist() == [[0, 3], [1, 99]]
  assert call(torch.tensor([3, 99], dtype=torch.int32)) == _lib.MTX_ERR_ARG and "not device memory" in _lib.last_error()
  torch.cuda.synchronize()


def test_slots_by_order_and_a_record_without_bits():
  seen, _ = record(5, 100)
  note(seen, None, 100, [7, 8, -1, 9], None, False)
  assert (seen.cpu() != 0).nonzero().tolist() == [[0, 7], [1, 8], [3, 9]]


@pytest.mark.parametrize("vocab", [256, 999, 1024])
@pytest.mark.parametrize("which", ["frequency", "presence"])
def test_infinite_penalties(vocab, which):
  """A token that was generated is out; the prompt's tokens and all others stay as they are."""
  b = Batch(6, vocab, history=0, biases=0, masks=0)
  prompt, new = list(range(0, vocab, 5)), list(range(3, vocab, 7))
  slots = b.seen.shape[0]
  note(b.seen, b.touched, vocab, prompt * slots, [s for s in range(slots) for _ in prompt], True)
  note(b.seen, b.touched, vocab, new * slots, [s for s in range(slots) for _ in new], False)
  b.keep[which][:] = float("inf")
  b.keep["presence" if which == "frequency" else "frequency"][:] = 0
  b.keep["repetition"][:] = 1
  out = torch.empty(6, vocab, device="cuda")
  b.run(out)
  want = b.logits.clone()
  want[:3, new] = want[4:, new] = float("-inf")  # (row 3 has no penalties)
  assert torch.equal(out, want)


@pytest.mark.parametrize("lists", [True, False])
def test_a_batch_without_any_bias(lists):
  """Lists of no entries at all, at addresses that nothing is read from, and no lists."""
  b = Batch(5, 700, biases=0)
  out = torch.full((5, 700), 9.0, device="cuda")
  if lists:
    nothing = torch.empty(4, dtype=torch.int32, device="cuda")[4:]  # (of its own an empty tensor has no address)
    place = nothing.untyped_storage().data_ptr()
    b.run(out, bias_token=place, bias_value=place)
  else:
    b.run(out, bias_off=None, bias_token=None, bias_value=None)
  close(out, b.want(), b)
