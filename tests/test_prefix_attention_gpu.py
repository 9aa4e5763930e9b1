"""Attention over shared prefixes against the definition in 64 bits."""

import ctypes
import math

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import draft_helpers as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_stalls():
  """No wait in the kernels has run out (their results would be wrong without an error)."""
  yield
  count = ctypes.c_uint32(1)
  _lib.check(_lib.load().mtx_prefix_attention_stalls(ctypes.byref(count)))
  assert count.value == 0


@pytest.fixture(autouse=True, params=[False, True], ids=["short", "long"])
def _page_map(request):
  """Page maps with room for the tokens there are, or for so many that prefixes of 64 pairs and more have the tensor cores."""
  Case.roomy = request.param


class Case:
  """Sequences with `rows` rows each; `lengths` tokens; `prefixes`: (first sequence, sequences, tokens) whose whole pages are shared and whose rest is a copy."""

  def __init__(self, rows, lengths, prefixes=(), heads=4, kv=2, dim=64, page=16, seed=0, lead=0, behind=0, spare=3, more_pages=0, spread=2.0, wide=0):
    g = torch.Generator().manual_seed(seed)
    self.heads, self.kv, self.dim, self.page = heads, kv, dim, page
    self.lengths, self.sequences = list(lengths), len(lengths)
    self.row0 = [lead]
    for n in rows:
      self.row0.append(self.row0[-1] + n)
    self.rows = self.row0[-1] + behind
    used = [-(-max(0, l) // page) for l in self.lengths]
    most = max(1, max(used, default=1)) + more_pages
    pairs, each = sum(rows) * heads // kv, max(1, len(prefixes))
    if self.roomy and prefixes and pairs >= 64 * each:
      most = max(most, int(600e6 / ((pairs - 128 / 5 * each * -(-pairs // (each * 128))) * kv * dim)) // page + 1)
    self.num_pages = sum(used) + spare
    order = torch.randperm(self.num_pages, generator=g).tolist()
    maps, at = torch.zeros(max(1, self.sequences), most, dtype=torch.int32), 0
    for s, n in enumerate(used):
      maps[s, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
      at += n
    k = torch.randn(kv, self.num_pages, page, dim, generator=g)
    v = torch.randn(kv, self.num_pages, page, dim, generator=g)
    for first, count, tokens in prefixes:
      whole = tokens // page
      for s in range(first + 1, first + count):
        maps[s, : min(whole, used[s])] = maps[first, : min(whole, used[s])]
        if tokens % page and used[s] > whole:
          k[:, maps[s, whole], : tokens % page] = k[:, maps[first, whole], : tokens % page]
          v[:, maps[s, whole], : tokens % page] = v[:, maps[first, whole], : tokens % page]
    self.bounds, self.prefix_len = [0], []
    for first, count, tokens in prefixes:
      while self.bounds[-1] < first:  # sequences that share nothing
        self.bounds.append(self.bounds[-1] + 1)
        self.prefix_len.append(0)
      self.bounds.append(first + count)
      self.prefix_len.append(tokens)
    self.prefixes = len(self.prefix_len)
    self.maps = maps
    self.k, self.v = k.to(torch.bfloat16).cuda(), v.to(torch.bfloat16).cuda()
    self.store = torch.full((max(1, self.rows), heads * dim + wide), 7.0, dtype=torch.bfloat16)
    self.store[:, : heads * dim] = spread * torch.randn(max(1, self.rows), heads * dim, generator=g)
    self.q = self.store.cuda()[:, : heads * dim]
    self.out = torch.full((max(1, self.rows), heads * dim + 2 * wide), 7.0, dtype=torch.bfloat16, device="cuda")[:, : heads * dim]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    self.dev = dict(row0=ints(self.row0), lengths=ints(self.lengths), page_map=maps.cuda(), prefix_seq0=ints(self.bounds), prefix_len=ints(self.prefix_len or [0]))
    self.scale = dim**-0.5
    self.need = _lib.load().mtx_prefix_attention_scratch_bytes(self.rows, self.sequences, self.prefixes, heads, kv, dim)
    self.scratch = torch.full((max(256, self.need),), 255, dtype=torch.uint8, device="cuda")  # (every word a NaN)

  def batch(self):
    d = {k: v.data_ptr() for k, v in self.dev.items()}
    if not self.prefixes:
      d["prefix_seq0"] = d["prefix_len"] = None
    return _lib.PrefixBatch(rows=self.rows, sequences=self.sequences, prefixes=self.prefixes, **d)

  def run(self, softcap=0.0, scratch=None, out=None, stream=None):
    out = self.out if out is None else out
    scratch = self.scratch if scratch is None else scratch
    _lib.check(_lib.load().mtx_prefix_attention(
        self.q.data_ptr(), self.q.stride(0), self.k.data_ptr(), self.v.data_ptr(), self.batch(), out.data_ptr(), out.stride(0), self.heads, self.kv, self.dim, self.num_pages, self.page,
        self.maps.shape[1], self.scale, softcap, scratch.data_ptr(), scratch.numel(), torch.cuda.current_stream().cuda_stream if stream is None else stream))
    return out

  def want(self, softcap=0.0):
    return ref.attention(self.q, self.k, self.v, self.row0, self.lengths, self.dev["page_map"], self.heads, self.scale, softcap)

  def check(self, softcap=0.0):
    got = self.run(softcap)
    want, bound = self.want(softcap)
    got = got.double().view(max(1, self.rows), self.heads, self.dim)[: want.shape[0]]
    there = ~want.isnan()
    off = ((got - want).abs() - bound)[there]
    assert off.numel() == 0 or float(off.max()) <= 0, (float(off.max()), int((off > 0).sum()), off.numel())
    assert bool((got[~there] == 7).all())  # rows that see nothing, or belong to nobody
    return got


@pytest.mark.parametrize("length", [1, 2, 7, 8, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 300, 1000, 4097])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_sequence(length, dim):
  Case([1], [length], dim=dim, seed=length).check()
  Case([min(4, length)], [length], dim=dim, seed=length, page=8).check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 1), (5, 1), (16, 1), (20, 4), (8, 8), (14, 2), (33, 3)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 8)])
def test_heads(heads, kv, dim, page):
  Case([1, 3, 2], [200, 333, 261], [(0, 3, 192)], heads=heads, kv=kv, dim=dim, page=page, seed=heads).check()
  Case([1, 5], [100, 70], heads=heads, kv=kv, dim=dim, page=page, seed=heads + 1).check()


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 8, 63, 64, 65, 100, 128, 200, 511, 1000])
def test_prefix_lengths(page, tokens):
  """Prefixes that end anywhere in a page or a tile."""
  Case([1, 2, 1, 4], [tokens + 1, tokens + 60, tokens + 129, tokens + 4], [(0, 4, tokens)], page=page, seed=tokens).check()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_of_a_prefix(dim):
  """More rows than a tile holds, tails from none to long ones."""
  g = torch.Generator().manual_seed(dim)
  rows = torch.randint(0, 9, (70,), generator=g).tolist()
  lengths = [700 + max(n, int(t)) for n, t in zip(rows, torch.randint(0, 300, (70,), generator=g))]
  Case(rows, lengths, [(0, 70, 700)], heads=10, kv=2, dim=dim, page=32, seed=dim).check()


def test_several_prefixes():
  g = torch.Generator().manual_seed(3)
  rows = torch.randint(1, 4, (24,), generator=g).tolist()
  of = [300] * 5 + [0] * 3 + [1100] * 10 + [64] * 2 + [0] * 4
  lengths = [p + n + int(t) for p, n, t in zip(of, rows, torch.randint(0, 200, (24,), generator=g))]
  Case(rows, lengths, [(0, 5, 300), (8, 10, 1100), (18, 2, 64)], heads=8, kv=2, dim=128, page=64, seed=5).check()


def test_rows_that_see_nothing():
  """Sequences without rows or tokens, rows in front of their sequence's first token, rows of nobody in front of the first sequence and behind the last."""
  Case([0, 2, 3, 1, 0], [50, 0, 2, 7, 0], lead=2, behind=5, seed=1).check()
  Case([2, 0, 6, 1, 1], [70, 100, 66, 90, 3], [(0, 5, 64)], lead=1, behind=200, heads=6, kv=3, seed=2).check()
  Case([3], [-4], seed=1).check()


def test_no_sequences():
  c = Case([1], [5])
  c.sequences = 0
  assert bool((c.run() == 7).all())
  c = Case([0, 0], [5, 9], [(0, 2, 4)], behind=3)
  assert bool((c.run() == 7).all())


def test_sequences_inside_a_prefix():
  """Rows whose position lies within the prefix, beside sequences that go on behind it."""
  Case([4, 2, 3, 1, 5], [130, 200, 60, 129, 140], [(0, 5, 129)], seed=4).check()
  Case([2, 2], [64, 65], [(0, 2, 64)], seed=4).check()


@pytest.mark.parametrize("softcap", [5.0, 30.0])
def test_softcap(softcap):
  for dim in (64, 128, 256):
    Case([2, 1, 3], [300, 258, 400], [(0, 3, 256)], dim=dim, seed=7, spread=6.0).check(softcap)


def test_peaky_scores():
  """Scores of some hundred: one key has it all, and it may come last."""
  for dim in (64, 128, 256):
    c = Case([1, 2, 1], [600, 700, 520], [(0, 3, 512)], dim=dim, seed=11, spread=60.0)
    c.check()


def test_pitches():
  Case([1, 4, 2], [100, 300, 212], [(0, 3, 96)], dim=128, wide=24, seed=6).check()
  c = Case([1, 4, 2], [100, 300, 212], [(0, 3, 96)], dim=64, wide=8, seed=6)
  c.check()
  base = c.out._base if c.out._base is not None else c.out
  assert bool((base[:, 256:] == 7).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_nobody_sees(dim, bad):
  """Whatever stands behind a sequence's tokens, in pages of nobody and in the later rows' own keys and values, changes nothing for the rows that do not see it."""
  c = Case([1, 4, 2, 1], [301, 333, 260, 257], [(0, 4, 250)], dim=dim, page=32, seed=dim, spare=9)
  clean = c.check().clone()
  for s in range(4):
    last = c.lengths[s] - 1
    page, at = int(c.maps[s, last // 32]), last % 32
    c.k[:, page, at + 1 :] = bad
    c.v[:, page, at + 1 :] = bad
  owned = set(c.maps.flatten().tolist())
  for page in range(c.num_pages):
    if page not in owned:
      c.k[:, page], c.v[:, page] = bad, bad
  assert torch.equal(c.check(), clean)
  # the last row of a sequence sees its own value, the rows in front of it do not
  for s, n in ((1, 4), (2, 2)):
    last = c.lengths[s] - 1
    c.v[:, int(c.maps[s, last // 32]), last % 32, ::3] = bad
  got = c.run().double().view(c.rows, c.heads, dim)
  mine = [c.row0[2] - 1, c.row0[3] - 1]
  others = [r for r in range(c.rows) if r not in mine]
  assert torch.equal(got[others], clean[others])
  for r in mine:
    assert not bool(got[r, :, ::3].isfinite().any()) and torch.equal(got[r, :, 1::3], clean[r, :, 1::3])


def test_numbers_that_a_prefix_has():
  """An infinite value or a NaN in a shared token reaches every row that sees it, and its channel alone."""
  c = Case([1, 2], [300, 310], [(0, 2, 256)], dim=64, seed=1)
  clean = c.check().clone()
  c.v[0, int(c.maps[0, 3]), 5, 7] = math.inf
  got = c.run().double().view(c.rows, c.heads, 64)
  assert bool(got[:, :2, 7].isinf().all())
  clean[:, :2, 7] = got[:, :2, 7]
  assert torch.equal(got, clean)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_that_are_none(dim):
  """A NaN in a shared key reaches all rows of its key head, wherever in a tile the token is, and no other head.  Keys far below all others weigh nothing."""
  rows = [4] * 32
  c = Case(rows, [600 + n for n in rows], [(0, 32, 512)], heads=8, kv=2, dim=dim, page=16, seed=dim)
  clean = c.check().clone()
  for token in (4, 5, 6, 7, 511):
    at = (1, int(c.maps[0, token // 16]), token % 16, 3)
    was = c.k[at].clone()
    c.k[at] = math.nan
    got = c.run().double().view_as(clean)
    c.k[at] = was
    assert bool(got[:, 4:].isnan().all()) and torch.equal(got[:, :4], clean[:, :4])
  c.q.abs_()
  clean = c.check().clone()
  for token in (4, 6, 63, 510):  # an infinite score: its weight is infinity over infinity
    at = (0, int(c.maps[0, token // 16]), token % 16, 9)
    was = c.k[at].clone()
    c.k[at] = math.inf
    got = c.run().double().view_as(clean)
    c.k[at] = was
    assert bool(got[:, :4].isnan().all()) and torch.equal(got[:, 4:], clean[:, 4:])
  c.k[:, c.maps[0, 2].long(), 1::2] = -1e30
  c.check()


@pytest.mark.parametrize("sequences", [2, 40])
def test_a_last_key_that_is_none(sequences):
  """A NaN in the one token that a sequence has behind the prefix: a part of its own whose only score is none."""
  c = Case([1] * sequences, [257] * sequences, [(0, sequences, 256)], heads=8, kv=2, dim=64, page=16)
  clean = c.check().clone()
  c.k[0, int(c.maps[1, 16]), 0, 9] = math.nan
  got = c.run().double().view_as(clean)
  assert bool(got[1, :4].isnan().all())
  clean[1, :4] = got[1, :4] = 0
  assert torch.equal(got, clean)


def test_sequences_that_descend():
  """Rows of two sequences at once would have more parts than the scratch has places: nothing is written."""
  c = Case([3] * 40, [200 + i for i in range(40)], [(0, 20, 64), (20, 20, 128)], heads=8, kv=2, dim=64, page=16)
  for name, at, to in (("row0", 7, 120), ("row0", 20, 120), ("prefix_seq0", 0, 30)):
    was = c.dev[name].clone()
    c.dev[name][at] = to
    c.out.fill_(7)
    assert bool((c.run() == 7).all())
    c.dev[name].copy_(was)
  c.check()


def test_pages_outside_the_pool():
  """They are read as page 0, and a length ends with the page map."""
  c = Case([1, 2], [90, 80], dim=64, page=16, seed=3)
  c.dev["page_map"][0, 2], c.dev["page_map"][1, 1] = -5, c.num_pages
  c.check()
  c.lengths[0] = 5000
  c.dev["lengths"][0] = 5000
  c.check()


def test_the_same_bits():
  """Every call, and every place of a sequence in the scratch, with whatever a scratch held."""
  c = Case([3, 1, 5, 2] * 8, [1100 + 37 * i for i in range(32)], [(0, 32, 1024)], heads=8, kv=2, dim=128, page=64, seed=5)
  first = c.run().clone()
  for fill in (0, 255, 127):
    c.scratch.fill_(fill)
    c.out.fill_(3)
    assert torch.equal(c.run(), first)


def test_streams_and_graphs():
  """Two captured calls with a scratch each, replayed at the same time on two streams while their lengths change."""
  cases = [Case([2, 1, 3], [400, 300, 350], [(0, 3, 256)], dim=128, page=32, seed=i, more_pages=2, spare=40) for i in range(2)]
  graphs, streams = [torch.cuda.CUDAGraph() for _ in cases], [torch.cuda.Stream() for _ in cases]
  torch.cuda.synchronize()
  for c, graph, stream in zip(cases, graphs, streams):
    with torch.cuda.graph(graph, stream=stream):
      c.run()
  for step in range(3):
    for c in cases:
      c.lengths = [l - 3 * step for l in c.lengths]
      c.dev["lengths"].copy_(torch.tensor(c.lengths, dtype=torch.int32))
      c.out.fill_(7)
    torch.cuda.synchronize()
    for _ in range(3):
      for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
          graph.replay()
    torch.cuda.synchronize()
    for c in cases:
      want, bound = c.want()
      assert bool(((c.out.double().view_as(want) - want).abs() <= bound).all())


def test_many_sequences():
  """More sequences than a CTA keeps entries of, with and without prefixes."""
  g = torch.Generator().manual_seed(8)
  rows = torch.randint(0, 3, (300,), generator=g).tolist()
  lengths = [40 + n + int(t) for n, t in zip(rows, torch.randint(0, 60, (300,), generator=g))]
  Case(rows, lengths, [(0, 100, 40), (150, 120, 33)], seed=8).check()
  Case(rows, lengths, seed=9).check()
  Case([1] * 128, [20] * 128, seed=10).check()
  Case([1] * 127, [50] * 127, [(0, 127, 32)], seed=11).check()


def test_far_pages():
  """A pool of more than 2^31 values, its ends in use."""
  kv, num_pages, page, dim = 2, 140000, 64, 128
  c = Case([2, 1], [200, 190], [(0, 2, 128)], kv=kv, dim=dim, page=page, seed=1)
  k, v = c.k, c.v
  c.k, c.v = (torch.zeros(kv, num_pages, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
  far = torch.arange(c.num_pages) * ((num_pages - 1) // (c.num_pages - 1)) + (num_pages - 1) % (c.num_pages - 1)
  c.k[:, far], c.v[:, far] = k, v
  c.maps = far[c.maps.long()].int()
  c.dev["page_map"].copy_(c.maps)
  c.num_pages = num_pages
  c.check()


def test_as_paged_attention():
  """One row per sequence and no prefix: what mtx_paged_attention gives, within both roundings."""
  lib = _lib.load()
  c = Case([1] * 6, [70, 1, 300, 129, 64, 500], heads=8, kv=2, dim=128, page=16, seed=2)
  c.scale = 1.0
  c.q.mul_(0.1)
  got = c.run().double()
  need = lib.mtx_paged_attention_scratch_bytes(6, 2, 8, 128, c.maps.shape[1] * 16)
  scratch, out = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(6, 1024, dtype=torch.bfloat16, device="cuda")
  _lib.check(lib.mtx_paged_attention(c.q.contiguous().data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.dev["lengths"].data_ptr(), c.dev["page_map"].data_ptr(), out.data_ptr(), 6, 8, 2, 128,
                                     c.num_pages, 16, c.maps.shape[1], 0.0, scratch.data_ptr(), torch.cuda.current_stream().cuda_stream))
  _, bound = c.want()
  assert bool(((out.double() - got).abs().view_as(bound) <= 2 * bound).all())


@pytest.mark.parametrize("dim,heads,kv", [(64, 20, 4), (128, 16, 4), (256, 8, 4), (128, 6, 1), (64, 32, 2)])
def test_long_prefixes(dim, heads, kv):
  """Many tiles of each item in a CTA, several items of it, halves that are not full; more than once, since what is not waited for may come in time by chance."""
  g = torch.Generator().manual_seed(heads)
  rows = torch.randint(1, 6, (48,), generator=g).tolist()
  c = Case(rows, [5001 + n + int(t) for n, t in zip(rows, torch.randint(0, 90, (48,), generator=g))], [(0, 48, 5001)], heads=heads, kv=kv, dim=dim, page=64, seed=dim)
  first = c.check()
  for _ in range(5):
    assert torch.equal(c.run().double().view_as(first), first)


@pytest.mark.parametrize("name,at,to", [("prefix_seq0", 0, 30), ("prefix_seq0", 1, 45), ("prefix_seq0", 2, 10), ("row0", 7, 120), ("row0", 39, 200), ("row0", 0, 500)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_short_sequences_that_descend(dim, name, at, to):
  """Tails of one tile, that no other part joins, are not written either, with the prefixes in a kernel of their own or not; what lies behind the last row or sequence descends too."""
  c = Case([3] * 40, [8 + i % 8 for i in range(40)], [(0, 20, 4), (20, 20, 3)], heads=8, kv=2, dim=dim, page=8, seed=dim)
  was = c.dev[name].clone()
  c.dev[name][at] = to
  assert bool((c.run() == 7).all())
  c.dev[name].copy_(was)
  c.check()


@pytest.mark.parametrize("dim,heads", [(64, 20), (128, 16), (256, 8)])
def test_behind_short_products(dim, heads):
  """Products of short sums in front, which start what comes next before they hold tensor memory of their own: every step ends, with the results that it has alone."""
  lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
  c = Case([5] * 40, [300 + i for i in range(40)], [(0, 40, 256)], heads=heads, kv=4, dim=dim, page=16, seed=dim)
  first = c.check()
  x, w = torch.randn(32, 128, device="cuda").to(torch.bfloat16), torch.randn(19200, 128, device="cuda").to(torch.bfloat16)
  ys = [torch.empty(32, 19200, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
  for _ in range(50):
    for y in ys:
      _lib.check(lib.mtx_linear(x.data_ptr(), w.data_ptr(), y.data_ptr(), 32, 19200, 128, 1, stream))
    c.run()
  assert torch.equal(c.out.double().view_as(first), first) and torch.equal(ys[0], ys[1])
  want = x.double() @ w.double().T
  assert bool(((ys[0].double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-13 * (x.double().abs() @ w.double().abs().T)).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("count", [129, 200, 300])
def test_many_sequences_of_few_prefixes(count, dim):
  """More sequences than a CTA keeps entries of, with the prefixes in a kernel of their own where the page map has room."""
  g = torch.Generator().manual_seed(count)
  rows = torch.randint(1, 4, (count,), generator=g).tolist()
  lengths = [150 + n + int(t) for n, t in zip(rows, torch.randint(0, 100, (count,), generator=g))]
  first = Case(rows, lengths, [(0, count, 150)], heads=8, kv=2, dim=dim, page=16, seed=count)
  got = first.check()
  for _ in range(3):
    assert torch.equal(first.run().double().view_as(got), got)
  Case(rows, lengths, [(0, 70, 100), (70, count - 70, 140)], heads=8, kv=2, dim=dim, page=16, seed=count + 1).check()
