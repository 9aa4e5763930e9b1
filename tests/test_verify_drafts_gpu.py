"""Verification of drafted tokens against the definition in 64 bits: the same tokens wherever no decision lies next to a border."""

import math

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import draft_helpers as ref

pytestmark = pytest.mark.gpu


class Case:

  def __init__(self, rows, vocab, draft=True, seed=0, heat=None, draft_heat=None, lead=0, behind=0, pitch=0, shift=0, spread=3.0, apart=0.7):
    g = torch.Generator().manual_seed(seed)
    self.vocab, self.sequences = vocab, len(rows)
    self.row0 = [lead]
    for n in rows:
      self.row0.append(self.row0[-1] + n)
    self.rows = self.row0[-1] + behind
    logits = spread * torch.randn(max(1, self.rows), vocab, generator=g)
    drafted = logits + apart * torch.randn(max(1, self.rows), vocab, generator=g)
    noise = -torch.log(-torch.log(torch.rand(max(1, self.rows), vocab, generator=g).clamp(1e-9, 1 - 1e-7)))
    self.token = torch.roll((drafted + noise).argmax(1), 1).int()
    self.heat = 0.5 + torch.rand(self.sequences, generator=g) if heat is None else torch.tensor(heat, dtype=torch.float32)
    self.draft_heat = None if draft_heat is None else torch.tensor(draft_heat, dtype=torch.float32)
    self.accept, self.pick = torch.rand(max(1, self.rows), generator=g), torch.rand(self.sequences, generator=g)
    self.pitch, self.shift = vocab + pitch, shift
    self.logits, self.drafted = logits, drafted if draft else None

  def put(self, t):
    store = torch.full((t.shape[0] * self.pitch + self.shift + 8,), 77.0, device="cuda")
    view = store[self.shift :].as_strided(t.shape, (self.pitch, 1), self.shift)
    view.copy_(t)
    return view

  def upload(self):
    self.dev = dict(row0=torch.tensor(self.row0, dtype=torch.int32).cuda(), token=self.token.cuda(), target=self.put(self.logits), temperature=self.heat.cuda(),
                    accept_u=self.accept.cuda(), pick_u=self.pick.cuda())
    if self.drafted is not None:
      self.dev["draft"] = self.put(self.drafted)
    if self.draft_heat is not None:
      self.dev["draft_temperature"] = self.draft_heat.cuda()
    self.accepted = torch.full((max(1, self.sequences),), -9, dtype=torch.int32, device="cuda")
    self.emitted = torch.full((max(1, self.rows),), -9, dtype=torch.int32, device="cuda")
    self.scratch = torch.full((max(16, _lib.load().mtx_verify_drafts_scratch_bytes(self.rows, self.sequences, self.vocab)),), 255, dtype=torch.uint8, device="cuda")

  def run(self):
    batch = _lib.DraftBatch(rows=self.rows, sequences=self.sequences, vocab=self.vocab, ld_target=self.pitch, ld_draft=self.pitch, **{k: v.data_ptr() for k, v in self.dev.items()})
    _lib.check(_lib.load().mtx_verify_drafts(batch, self.accepted.data_ptr(), self.emitted.data_ptr(), self.scratch.data_ptr(), self.scratch.numel(), torch.cuda.current_stream().cuda_stream))

  def compare(self, near_most=None, **close):
    heat = self.heat.double()
    want = ref.verified(self.logits, self.drafted, self.row0, self.token, heat, heat if self.draft_heat is None else self.draft_heat.double(), self.accept.double(), self.pick.double(), self.vocab, **close)
    accepted, emitted = self.accepted.tolist(), self.emitted.tolist()
    skipped = 0
    for s, (kept, tokens, near, (low, high)) in enumerate(want):
      if near:
        skipped += 1
        continue
      got = emitted[self.row0[s] : self.row0[s + 1]]
      assert accepted[s] == kept and got[:kept] == tokens[:kept] and got[kept + 1 :] == tokens[kept + 1 :], (s, accepted[s], kept, got, tokens)
      assert not got or low <= got[kept] <= high, (s, got[kept], low, high)
      drawn = got[kept] if got else -1
      if drawn >= 0 and self.heat[s] > 0:  # (never a token that the target may not say)
        assert not float(self.logits[self.row0[s] + kept, drawn]) in (-math.inf, math.nan)
    assert skipped <= (self.sequences // 50 if near_most is None else near_most)
    assert all(t == -9 for t in emitted[: self.row0[0]] + emitted[self.row0[-1] :] if self.rows)
    return want

  def check(self, **more):
    self.upload()
    self.run()
    return self.compare(**more)


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 33, 255, 1000, 1024, 1025, 4095, 4097, 32768, 50001])
@pytest.mark.parametrize("draft", [True, False])
def test_vocabularies(vocab, draft):
  c = Case([5, 1, 3, 2, 8], vocab, draft, seed=vocab)
  c.check(near_most=0)


@pytest.mark.parametrize("draft", [True, False])
def test_many_sequences(draft):
  """Drafts that stay, that do not, and how far each sequence comes."""
  want = Case([1 + i % 6 for i in range(200)], 700, draft, seed=5, spread=2.0, apart=0.4).check()
  kept = {w[0] for w in want}
  assert 0 in kept and (not draft or max(kept) >= 4)


def test_the_expanded_vocabulary():
  Case([5, 3], 264192, True, seed=1).check()
  Case([2, 4], 264192, False, seed=2).check()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("rows,vocab,pitch,shift", [([5] * 7 + [1], 264192, 0, 0), ([5] * 7 + [1], 262147, 1, 3), ([3, 2, 4], 786433, 3, 2), ([2, 3, 3], 1000003, 0, 1)])
def test_much_to_read(rows, vocab, pitch, shift, draft):
  """Chunks of 4096 tokens; greedy sequences beside others, masked logits and rows that leave one token."""
  c = Case(rows, vocab, draft, seed=vocab, pitch=pitch, shift=shift, heat=[0.9, 0.0, 1.1] + [0.7] * (len(rows) - 3))
  c.logits[c.row0[0], : vocab - 9000] = -math.inf
  last = c.row0[-1] - 1
  c.logits[last, :] = -math.inf
  c.logits[last, vocab // 2] = 1.0
  want = c.check()
  assert want[-1][1][-1] in (vocab // 2, -1)


@pytest.mark.parametrize("pitch,shift", [(0, 1), (1, 0), (3, 2), (5, 3), (4, 4)])
def test_places(pitch, shift):
  Case([4, 2, 3], 9001, True, seed=pitch, pitch=pitch, shift=shift).check(near_most=0)


def test_greedy():
  """Temperature 0: the largest logit, of equal ones the first; beside sequences that draw."""
  for draft in (True, False):
    c = Case([4] * 12, 3000, draft, seed=4, heat=[0.0, 0.8] * 6)
    c.logits[:, 100] = c.logits[:, 2500] = 20.0
    for s in range(0, 12, 2):
      for i in range(s // 4):
        c.token[c.row0[s] + 1 + i] = 100
    c.token[c.row0[6] + 1] = 2500  # as large, but not the first
    want = c.check(near_most=0)
    assert want[2][0] == 0 and want[4][0] == 1 and want[8][0] == 2 and want[0][1][0] == 100


def test_sure_drafts():
  """A draft temperature of 0 is a draft without probabilities."""
  c = Case([3] * 8, 500, True, seed=2, draft_heat=[0.0, 0.7] * 4)
  c.check(near_most=0)


def test_the_drafts_own_temperature():
  Case([4] * 10, 500, True, seed=3, draft_heat=[0.3 + 0.2 * i for i in range(10)]).check(near_most=0)


@pytest.mark.parametrize("draft", [True, False])
def test_masks(draft):
  """Masked logits on either side; rows that leave one token, and rows that leave none."""
  c = Case([4, 4, 4, 4, 4, 1], 2049, draft, seed=6)
  c.logits[c.row0[0] : c.row0[1], :1500] = -math.inf
  one = torch.full((4, 2049), -math.inf)
  one[:, 77] = 1.0
  c.logits[c.row0[1] : c.row0[2]] = one
  c.token[c.row0[1] + 1 : c.row0[2]] = 77
  c.logits[c.row0[2]] = -math.inf
  c.token[c.row0[3] + 1] = 5
  c.logits[c.row0[3], 5] = -math.inf
  c.logits[c.row0[5]] = -math.inf
  if draft:
    c.drafted[c.row0[4]] = -math.inf
    c.drafted[c.row0[3], :1000] = -math.inf
  want = c.check(near_most=0)
  assert want[2][1] == [-1, -1, -1, -1] and want[5][1] == [-1]
  assert draft or want[1][0] == 3


def test_logits_that_are_no_numbers():
  for draft in (True, False):
    c = Case([3, 3, 3, 2], 1500, draft, seed=8, heat=[1.0, 0.0, 0.7, 1.0])
    c.logits[c.row0[0], 3], c.logits[c.row0[1], 4], c.logits[c.row0[2], 9] = math.nan, math.nan, math.inf
    c.logits[c.row0[3]] = math.nan
    if draft:
      c.drafted[c.row0[0], 8], c.drafted[c.row0[2], 9] = math.nan, math.inf
    want = c.check(near_most=0)
    assert want[3][1] == [-1, -1]


def test_equal_probabilities():
  """Drafts of the target itself: accept_u < 1 keeps every one."""
  c = Case([6] * 20, 900, True, seed=9, apart=0.0)
  c.upload()
  c.run()
  assert c.accepted.tolist() == [5] * 20


def test_ends_of_the_numbers():
  """0 keeps what the target may say, and draws the first token that it may say; numbers next to 1 draw the last one at most."""
  c = Case([3] * 4, 2000, True, seed=10)
  c.logits[:, :7], c.logits[:, 1990:] = -math.inf, -math.inf
  c.drafted = torch.where(c.logits == -math.inf, -math.inf, c.drafted)
  c.accept[:] = 0
  c.pick[:2], c.pick[2:] = 0, 1 - 2.0**-24
  for s in range(4):
    c.token[c.row0[s] + 1 : c.row0[s + 1]] = 1000
  c.upload()
  c.run()
  assert c.accepted.tolist() == [2] * 4
  got = c.emitted.view(4, 3)[:, 2].tolist()
  assert got[:2] == [7, 7] and all(1500 < t < 1990 for t in got[2:])


def test_drafts_outside_the_vocabulary():
  for draft in (True, False):
    c = Case([3, 3, 3], 800, draft, seed=11)
    c.token[c.row0[0] + 1], c.token[c.row0[1] + 1], c.token[c.row0[2] + 1] = -1, 800, 2**31 - 1
    want = c.check(near_most=0)
    assert [w[0] for w in want] == [0, 0, 0]


def test_rows_of_nobody():
  c = Case([0, 3, 0, 2, 0], 600, True, seed=12, lead=3, behind=4)
  want = c.check(near_most=0)
  assert c.accepted.tolist()[0] == 0 and want[0][1] == []
  c = Case([0, 0], 600, False, seed=12)
  c.upload()
  c.run()
  assert c.accepted.tolist() == [0, 0]


def test_peaky_logits():
  """Logits of some thousand over a low temperature."""
  Case([4] * 6, 5000, True, seed=13, spread=1000.0, apart=1.0, heat=[0.05] * 6).check(near_most=0)


def test_flat_logits():
  """All tokens alike, weights of 1 each: their number decides, whole numbers have no rounding."""
  c = Case([2] * 6, 100000, False, seed=14, spread=0.0)
  c.check(near_most=0, close=2.0**-40)


def test_the_distribution():
  """Whatever the draft, the first emitted token is distributed as the target says: 6000 sequences of one draft each, within five standard deviations."""
  vocab, many = 5, 6000
  g = torch.Generator().manual_seed(1)
  target, draft = torch.tensor([1.0, 0.2, -0.5, 0.4, -1.0]), torch.tensor([-1.0, 0.9, 0.5, 0.4, 0.3])
  c = Case([2] * many, vocab, True, seed=15, heat=[1.0] * many)
  c.logits[:], c.drafted[:] = target, draft
  c.token[1::2] = torch.multinomial(torch.softmax(draft, 0), many, True, generator=g).int()
  c.upload()
  c.run()
  first = c.emitted.view(many, 2)[:, 0].long().cpu()
  p = torch.softmax(target, 0)
  share = torch.bincount(first, minlength=vocab) / many
  assert bool(((share - p).abs() <= 5 * (p * (1 - p) / many).sqrt()).all())


def test_the_same_every_time():
  c = Case([5] * 30, 20001, True, seed=16)
  c.upload()
  c.run()
  first = c.accepted.clone(), c.emitted.clone()
  for fill in (0, 255):
    c.scratch.fill_(fill)
    c.run()
    assert torch.equal(c.accepted, first[0]) and torch.equal(c.emitted, first[1])


def test_streams_and_graphs():
  """Two captured calls with a scratch each, replayed at the same time on two streams over new logits and numbers."""
  cases = [Case([3] * 20, 6001, i == 0, seed=20 + i) for i in range(2)]
  graphs, streams = [torch.cuda.CUDAGraph() for _ in cases], [torch.cuda.Stream() for _ in cases]
  for c in cases:
    c.upload()
  torch.cuda.synchronize()
  for c, graph, stream in zip(cases, graphs, streams):
    with torch.cuda.graph(graph, stream=stream):
      c.run()
  for step in range(3):
    for i, c in enumerate(cases):
      n = Case([3] * 20, 6001, i == 0, seed=30 + 2 * step + i)
      for name in ("logits", "drafted", "token", "heat", "accept", "pick"):
        setattr(c, name, getattr(n, name))
      n.upload()
      for k, v in c.dev.items():
        v.copy_(n.dev[k])
    torch.cuda.synchronize()
    for _ in range(2):
      for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
          graph.replay()
    torch.cuda.synchronize()
    for c in cases:
      c.compare(near_most=0)


def test_rows_far_apart():
  """Logits more than 2^31 apart."""
  vocab, rows = 3000, 3
  c = Case([rows], vocab, False, seed=17)
  c.pitch = (1 << 30) + 5
  c.put = lambda t: _far(t, c.pitch)
  c.check(near_most=0)


def _far(t, pitch):
  store = torch.empty(pitch * (t.shape[0] - 1) + t.shape[1], device="cuda")
  view = store.as_strided(t.shape, (pitch, 1))
  view.copy_(t)
  return view


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("heat,size", [(1.0, s) for s in (1e6, 1e7, 1e8, 3e8, 7e8, 1.5e9, 3e9, 1e10, 2e10, 1e15, 1e20, 1e30, 1e38)]
                         + [(2.0**-20, s) for s in (20.0, 100.0, 700.0, 1000.0, 2900.0, 5000.0, 1e5)] + [(1e-6, 4000.0), (0.01, 1e8)])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_logits_over_low_temperatures(heat, size, sign, draft):
  """From where all tokens next to the largest count to where it alone does: exponents of 2^20 to infinity, either sign."""
  c = Case([4, 3, 5, 2, 1, 6], 1500, draft, seed=23, heat=[heat] * 6)
  g = torch.Generator().manual_seed(int(size) % 1000)
  tops = 1200 + torch.randperm(200, generator=g)[:40]
  own = torch.arange(1000, 1010)  # tokens of the draft's alone
  for part, best_of in ((c.logits, tops),) + (((c.drafted, torch.cat([tops[:10], own, tops[10:25]])),) if draft else ()):
    part.copy_(sign * size * (1 - 0.25 * sign * torch.rand(part.shape, generator=g)))
    best = part.amax(1) + 0.05 * size
    part[:, best_of] = best[:, None]
    for i, t in enumerate(best_of[-15:].tolist() if part is c.drafted else best_of[10:].tolist()):  # up to five steps below the largest
      for _ in range(i % 6):
        part[:, t] = torch.nextafter(part[:, t], torch.tensor(-math.inf))
  c.token = torch.cat([tops[:10], own])[torch.randint(0, 20, (c.rows,), generator=g)].int()
  c.upload()
  c.run()
  want = c.compare(near_most=1)
  assert all(t >= 0 for w in want for t in w[1][: w[0] + 1])
  assert all(t in tops.tolist() for t in c.emitted.tolist() if t != -1)


@pytest.mark.parametrize("left", [1e-2, 1e-4, 1e-6, 1e-7])
def test_what_a_draft_leaves_of_its_target(left):
  """A draft that has one token more, whose share is `left`: of all others the same part is left, so that they are drawn by their own weights, within 2^-19 of their sum (weights off by 2^-20.5, a
  thread's sums of up to 16 of them by 2^-20)."""
  c = Case([2] * 300, 3000, True, seed=24, heat=[1.0] * 300, spread=2.0)
  c.logits[:, 2000], c.logits[:, 700] = 8.0, -math.inf
  c.drafted.copy_(c.logits)
  c.drafted[:, 700] = math.log(left) + torch.logsumexp(c.logits, 1)
  c.token[:] = 700
  c.upload()
  c.run()
  assert c.accepted.tolist() == [0] * 300
  for s, drawn in enumerate(c.emitted[::2].tolist()):
    up = c.logits[2 * s].double().exp().cumsum(0)
    want = float(c.pick[s]) * float(up[-1])
    low, high = (float(up[drawn - 1]) if drawn > 0 else 0.0) - 2.0**-19 * float(up[-1]), float(up[drawn]) + 2.0**-19 * float(up[-1])
    assert low <= want <= high and drawn != 700, (s, drawn, want / float(up[-1]), low / float(up[-1]), high / float(up[-1]))


@pytest.mark.parametrize("apart", [1e-1, 1e-2, 1e-3, 1e-4, 1e-5])
def test_drafts_next_to_their_target(apart):
  """Drawn from a difference that is small beside the target: a border lies within 2^-18.5 of the target's whole sum.  (Weights are off by 2^-20.5 of themselves, and so are both whole sums: of the
  target's part of a sum once that, of the draft's part three times.)"""
  c = Case([2] * 40, 32768, True, seed=25, heat=[1.0] * 40, apart=apart)
  c.accept[:] = 1 - 2.0**-24
  p, q = (torch.softmax(x.double(), 1) for x in (c.logits, c.drafted))
  token = torch.where(p > 1e-6, q / p, 0.0).argmax(1)  # the one that the draft says most too often
  c.token[1::2] = token[::2].int()
  c.upload()
  c.run()
  assert c.accepted.tolist() == [0] * 40
  for s, drawn in enumerate(c.emitted[::2].tolist()):
    weight = (p[2 * s] - q[2 * s]).clamp(min=0)
    up = weight.cumsum(0)
    want = float(c.pick[s]) * float(up[-1])
    assert (float(up[drawn - 1]) if drawn > 0 else 0.0) - 2.0**-18.5 <= want <= float(up[drawn]) + 2.0**-18.5
    assert abs(float(weight[drawn])) > 0 or float(q[2 * s, drawn] - p[2 * s, drawn]) < 2.0**-18.5 * float(p[2 * s, drawn])
