"""Draws from logits behind masks: rows that a mask empties, masks that leave fewer tokens than a strategy keeps."""

import pytest
import torch

from maxtext_indextts2_b200 import _lib

pytestmark = pytest.mark.gpu

STRATEGIES = ["greedy", "weighted", "nucleus", "topk"]


def stream():
  return torch.cuda.current_stream().cuda_stream


def masked(logits, allowed):
  """logits [rows, vocab] behind the masks allowed [rows, vocab], by the entry point, in place."""
  rows, vocab = logits.shape
  words = -(-vocab // 32)
  bits = torch.zeros(rows, words * 32, dtype=torch.int64)
  bits[:, :vocab] = allowed
  mask = (bits.view(rows, words, 32) << torch.arange(32)).sum(-1).to(torch.int32).cuda()
  c = _lib.LogitControls(allowed_rows=rows, allowed=mask.data_ptr(), ld_allowed=words)
  _lib.check(_lib.load().mtx_control_logits(logits.data_ptr(), vocab, logits.data_ptr(), vocab, rows, vocab, c, stream()))
  torch.cuda.synchronize()  # (the mask is the caller's until then)


def drawn(logits, strategy, seed=7, top_k=50, nucleus_p=0.9, temperature=0.8):
  rows, vocab = logits.shape
  rng = torch.tensor([3, seed, 1, 0], dtype=torch.int32, device="cuda")
  scratch = torch.empty(5 * rows, device="cuda")
  token, log_prob = torch.full((rows,), -9, dtype=torch.int32, device="cuda"), torch.full((rows,), 9.0, device="cuda")
  _lib.check(_lib.load().mtx_sample_rows(logits.data_ptr(), rows, vocab, vocab, _lib.SAMPLING[strategy], top_k, nucleus_p, temperature, rng.data_ptr(), 0, scratch.data_ptr(),
                                         token.data_ptr(), log_prob.data_ptr(), stream()))
  return token, log_prob


@pytest.mark.parametrize("strategy", STRATEGIES)
@pytest.mark.parametrize("vocab", [1, 40, 3001])
def test_a_row_that_its_mask_empties(strategy, vocab):
  """It gives token -1 and log-probability -infinity and leaves the record as it was; its neighbours draw from what their masks leave."""
  g = torch.Generator().manual_seed(vocab)
  allowed = torch.zeros(5, vocab, dtype=torch.bool)
  allowed[0] = True
  allowed[2, torch.randperm(vocab, generator=g)[:3]] = True  # fewer than the 50 that top-k keeps
  allowed[4, vocab - 1] = True
  before = 3 * torch.randn(5, vocab, generator=g)
  logits = before.cuda()
  masked(logits, allowed)
  token, log_prob = drawn(logits, strategy)
  want = torch.log_softmax(torch.where(allowed, before.double(), float("-inf")), -1)
  for r in (0, 2, 4):
    t = int(token[r])
    assert 0 <= t < vocab and bool(allowed[r, t])
    # In units of 2^-24: a sum of vocab terms is off by vocab of itself at most, its exponentials by 4, their arguments (up to 32 in size) by 32; the logarithm
    # (up to 16) by 2 * 16, its sum with the maximum (up to 16) by 16, the last difference (up to 32) by 32.
    assert abs(float(log_prob[r]) - float(want[r, t])) <= (vocab + 4 + 32 + 32 + 16 + 32) * 2.0**-24
  for r in (1, 3):
    assert int(token[r]) == -1 and float(log_prob[r]) == float("-inf")
  pitch = -(-vocab // 8) * 8
  seen, touched = torch.zeros(5, pitch, dtype=torch.int16, device="cuda"), torch.zeros(5, -(-vocab // 256), dtype=torch.int32, device="cuda")
  _lib.check(_lib.load().mtx_note_tokens(seen.data_ptr(), pitch, touched.data_ptr(), touched.stride(0), 5, vocab, token.data_ptr(), None, 5, 0, stream()))
  assert seen.cpu().nonzero().tolist() == [[r, int(token[r])] for r in (0, 2, 4)] and touched.cpu().count_nonzero(1).tolist() == [1, 0, 1, 0, 1]


@pytest.mark.parametrize("strategy", STRATEGIES)
def test_a_row_of_nan(strategy):
  logits = torch.full((2, 300), float("nan"), device="cuda")
  logits[1] = torch.arange(300.0) % 7
  token, log_prob = drawn(logits, strategy)
  assert int(token[0]) == -1 and float(log_prob[0]) == float("-inf")
  assert 0 <= int(token[1]) < 300 and -20 < float(log_prob[1]) < 0


@pytest.mark.parametrize("strategy", STRATEGIES)
@pytest.mark.parametrize("low", [-2.0e7, -3.0e38])
def test_what_a_mask_leaves_may_be_very_low(strategy, low):
  """Allowed logits far below the value that a nucleus gives to what it cuts: no token that the mask forbids is drawn in their place."""
  vocab = 700
  allowed = torch.zeros(40, vocab, dtype=torch.bool)
  allowed[:, 100:600:7] = True
  logits = torch.full((40, vocab), low, device="cuda")
  logits[:, 350] = low * 0.99  # (100 + 7 * 35 + 5: not allowed)
  masked(logits, allowed)
  token, log_prob = drawn(logits, strategy, temperature=1.0)
  assert all(bool(allowed[r, t]) for r, t in enumerate(token.tolist()))
  assert bool(log_prob.isfinite().all())
