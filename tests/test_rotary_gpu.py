"""Rotary positions and the way into the pages against the definition in 64 bits."""

import ctypes
import math

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import draft_helpers as ref

pytestmark = pytest.mark.gpu

CODE = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
BF16, F32 = torch.bfloat16, torch.float32


def close(got, want, size, amplitude, far=0):
  """Angles in 64 bits (their reduced value rounded to 32), cosine and sine within two last bits, three roundings, then the result's own."""
  slack = (2.0**-20 + far * 2.0**-50) * abs(amplitude) * size
  return bool(((got.double() - want).abs() <= slack + ref.EPS[got.dtype] * (want.abs() + slack) + 2.0**-133).all())


class Case:

  def __init__(self, rows, heads, kv, dim, rot, half, ti=BF16, to=BF16, seed=0, base=10000.0, amplitude=1.0, most=4000, page=16, shift=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    self.rows, self.heads, self.kv, self.dim, self.rot, self.half, self.ti, self.to, self.amplitude, self.page = rows, heads, kv, dim, rot, half, ti, to, amplitude, page
    wide = (heads + 2 * kv) * dim
    self.ld = wide + extra
    store = torch.randn(rows * self.ld + shift, generator=g).to(ti)
    self.store = store.cuda()
    self.x = store[shift:].as_strided((rows, wide), (self.ld, 1), shift)
    self.at = self.store.data_ptr() + shift * self.store.element_size()
    self.freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    self.freq_dev = self.freq.cuda()
    self.pos = torch.randint(0, most, (rows,), generator=g).int()
    self.pos_dev = self.pos.cuda()
    self.q = torch.full((rows, heads * dim + extra), 7.0, dtype=to, device="cuda")
    self.k = torch.full((rows, kv * dim + extra), 7.0, dtype=to, device="cuda")

  def batch(self, **more):
    size = self.store.element_size()
    wide, kv_wide = self.heads * self.dim, self.kv * self.dim
    fields = dict(rows=self.rows, heads=self.heads, kv_heads=self.kv, dim=self.dim, rot_dims=self.rot, rot_half=int(self.half), amplitude=self.amplitude, type=CODE[self.ti],
                  out_type=CODE[self.to], freq=self.freq_dev.data_ptr(), pos=self.pos_dev.data_ptr(), q=self.at, ldq=self.ld, k=self.at + wide * size, ldk=self.ld,
                  v=self.at + (wide + kv_wide) * size, ldv=self.ld, q_out=self.q.data_ptr(), ldq_out=self.q.stride(0), k_out=self.k.data_ptr(), ldk_out=self.k.stride(0))
    return _lib.RotaryBatch(**{**fields, **more})

  def want(self):
    x = self.x.reshape(self.rows, -1, self.dim)
    turned = ref.rotated(x[:, : self.heads + self.kv], self.pos, self.freq, self.amplitude, self.half)
    size = x[:, : self.heads + self.kv].double().abs().amax(2, keepdim=True).expand_as(turned) * 2
    return turned[:, : self.heads], turned[:, self.heads :], x[:, self.heads + self.kv :].double(), size[:, : self.heads], size[:, self.heads :]


def run(batch, stream=None):
  _lib.check(_lib.load().mtx_rotary(batch, torch.cuda.current_stream().cuda_stream if stream is None else stream))


@pytest.mark.parametrize("rows,heads,kv,dim,rot", [(1, 1, 1, 2, 2), (5, 20, 4, 64, 64), (3, 16, 4, 128, 64), (2, 8, 4, 256, 256), (7, 3, 1, 80, 32), (4, 5, 5, 128, 50), (2, 2, 1, 1024, 1024), (9, 1, 0, 64, 0),
                                                   (3, 0, 2, 64, 64), (3, 4, 2, 33, 16), (130, 6, 2, 96, 96)])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("types", [(BF16, BF16), (F32, BF16), (F32, F32), (BF16, F32)])
def test_layouts(rows, heads, kv, dim, rot, half, types):
  c = Case(rows, heads, kv, dim, rot, half, *types, seed=rows * dim + rot, amplitude=1.25)
  run(c.batch())
  q, k, _, qs, ks = c.want()
  assert close(c.q.cpu().view(rows, heads, dim), q, qs, 1.25) and close(c.k.cpu().view(rows, kv, dim), k, ks, 1.25)


@pytest.mark.parametrize("rows,heads,kv,dim,rot,half", [(5000, 1, 1, 1024, 1024, True), (9000, 1, 1, 64, 64, True), (12001, 2, 1, 32, 20, False), (4500, 3, 2, 128, 64, True)])
def test_many_tokens(rows, heads, kv, dim, rot, half):
  """As many of a CTA as it takes, in one wave and in several, with the largest of cosines and sines."""
  c = Case(rows, heads, kv, dim, rot, half, seed=rows)
  run(c.batch())
  q, k, _, qs, ks = c.want()
  assert close(c.q.cpu().view(rows, heads, dim), q, qs, 1.0) and close(c.k.cpu().view(rows, kv, dim), k, ks, 1.0)


@pytest.mark.parametrize("shift,extra", [(1, 0), (0, 3), (3, 5), (8, 8)])
def test_places(shift, extra):
  for half in (False, True):
    c = Case(6, 4, 2, 64, 48, half, seed=shift, shift=shift, extra=extra)
    run(c.batch())
    q, k, _, qs, ks = c.want()
    assert close(c.q.cpu()[:, :256].reshape(6, 4, 64), q, qs, 1) and close(c.k.cpu()[:, :128].reshape(6, 2, 64), k, ks, 1)
    assert bool((c.q[:, 256:].float() == 7).all()) and bool((c.k[:, 128:].float() == 7).all())


@pytest.mark.parametrize("ti", [BF16, F32])
def test_far_positions(ti):
  """Positions up to 2^31 - 1, negative ones too (a turn back): 64-bit angles."""
  c = Case(40, 2, 1, 64, 64, True, ti, F32, seed=3)
  c.pos = torch.cat([torch.tensor([0, 1, -1, 2**31 - 1, -(2**31)]), torch.randint(-(2**31), 2**31, (35,), generator=torch.Generator().manual_seed(1))]).int()
  c.pos_dev = c.pos.cuda()
  run(c.batch())
  q, k, _, qs, ks = c.want()
  assert close(c.q.cpu().view(40, 2, 64), q, qs, 1, far=2**31) and close(c.k.cpu().view(40, 1, 64), k, ks, 1, far=2**31)


def test_there_and_back():
  c = Case(8, 4, 4, 64, 64, False, F32, F32, seed=8)
  run(c.batch())
  c.pos_dev.neg_()
  run(c.batch(q=c.q.data_ptr(), ldq=c.q.stride(0), k=c.k.data_ptr(), ldk=c.k.stride(0)))  # in place
  x = c.x.view(8, -1, 64)
  assert bool((c.q.cpu().view(8, 4, 64) - x[:, :4]).abs().max() < 2.0**-17) and bool((c.k.cpu().view(8, 4, 64) - x[:, 4:8]).abs().max() < 2.0**-17)


@pytest.mark.parametrize("half,dim,rot", [(False, 64, 64), (True, 64, 64), (True, 96, 34), (False, 33, 32)])
def test_in_place(half, dim, rot):
  c = Case(5, 3, 2, dim, rot, half, seed=dim)
  q, k, v, qs, ks = c.want()
  wide, size = 3 * dim, 2
  run(c.batch(q_out=c.at, ldq_out=c.ld, k_out=c.at + wide * size, ldk_out=c.ld))
  got = c.store.cpu().view(5, -1, dim)
  assert close(got[:, :3], q, qs, 1) and close(got[:, 3:5], k, ks, 1) and torch.equal(got[:, 5:].double(), v)


@pytest.mark.parametrize("dim,rot,page,kv", [(64, 64, 16, 4), (128, 64, 8, 2), (80, 20, 1, 1), (256, 256, 64, 8)])
@pytest.mark.parametrize("ti", [BF16, F32])
def test_pages(dim, rot, page, kv, ti):
  """Rows of several groups over scattered pages, rows of nobody among them, pages that are not there; everything else in the pools stays."""
  g = torch.Generator().manual_seed(dim + page)
  rows, groups, most, num_pages = 50, 4, 7, 40
  c = Case(rows, 2 * kv, kv, dim, rot, True, ti, BF16, seed=page)
  group = torch.randint(-1, groups + 1, (rows,), generator=g).int()
  seen, pos = set(), []
  for r in range(rows):
    while True:
      p = int(torch.randint(-2, most * page + 2, (1,), generator=g))
      if (int(group[r]), p) not in seen:
        break
      if len(seen) > groups * most * page // 2:
        p = -1
        break
    seen.add((int(group[r]), p))
    pos.append(p)
  c.pos = torch.tensor(pos, dtype=torch.int32)
  c.pos_dev = c.pos.cuda()
  page_map = torch.randperm(num_pages, generator=g)[: groups * most].int().view(groups, most)
  page_map[1, 2], page_map[2, 0] = -1, num_pages
  kp = torch.randn(kv, num_pages, page, dim, generator=g).to(BF16)
  vp = torch.randn(kv, num_pages, page, dim, generator=g).to(BF16)
  kd, vd, gd, md = kp.cuda(), vp.cuda(), group.cuda(), page_map.cuda()
  pages = dict(k_pages=kd.data_ptr(), v_pages=vd.data_ptr(), groups=groups, num_pages=num_pages, tokens_per_page=page, max_pages_per_group=most, group=gd.data_ptr(), page_map=md.data_ptr())
  run(c.batch(k_out=None, **pages))
  q, k, v, qs, ks = c.want()
  got = c.q.cpu().view(rows, 2 * kv, dim)
  want_k, want_v, slack = kp.double(), vp.double(), torch.zeros_like(kp, dtype=torch.float64)
  for r in range(rows):
    mine = 0 <= int(group[r]) < groups and pos[r] >= 0
    if not mine:
      assert bool((got[r].float() == 7).all())
      continue
    assert close(got[r : r + 1], q[r : r + 1], qs[r : r + 1], 1)
    at = int(page_map[group[r], pos[r] // page]) if pos[r] // page < most else -1
    if 0 <= at < num_pages:
      want_k[:, at, pos[r] % page], want_v[:, at, pos[r] % page], slack[:, at, pos[r] % page] = k[r], v[r].to(BF16).double(), ks[r]
  assert torch.equal(vd.cpu().double(), want_v) and close(kd.cpu(), want_k, slack, 1) is True
  same = slack == 0
  assert torch.equal(kd.cpu()[same], kp[same])


def test_group_of_each_row():
  """Without group, row r is page group r; keys to rows of their own at the same time."""
  c = Case(3, 2, 1, 64, 64, True, seed=1, most=16)
  pool = torch.zeros(1, 4, 16, 64, dtype=BF16, device="cuda")
  values = torch.zeros_like(pool)
  page_map = torch.tensor([[2], [0], [3]], dtype=torch.int32, device="cuda")
  run(c.batch(k_pages=pool.data_ptr(), v_pages=values.data_ptr(), groups=3, num_pages=4, tokens_per_page=16, max_pages_per_group=1, page_map=page_map.data_ptr()))
  for r, at in enumerate((2, 0, 3)):
    assert torch.equal(pool[0, at, int(c.pos[r])], c.k[r]) and torch.equal(values[0, at, int(c.pos[r])].cpu(), c.x[r, 192:])


def test_values_that_are_no_numbers():
  c = Case(2, 1, 1, 64, 32, True, F32, F32, seed=1)
  c.store[3], c.store[40] = math.nan, math.inf
  run(c.batch())
  q = c.q.cpu()
  assert bool(q[0, 3].isnan()) and bool(q[0, 19].isnan()) and bool(q[0, 40].isinf()) and int(q.isfinite().logical_not().sum()) == 3


def test_far_pages():
  """A pool of more than 2^31 values."""
  page, dim, num_pages = 64, 128, 300000
  pool, values = torch.empty(1, num_pages, page, dim, dtype=BF16, device="cuda"), torch.empty(1, num_pages, page, dim, dtype=BF16, device="cuda")
  c = Case(2, 1, 1, dim, dim, True, seed=2, most=64)
  page_map = torch.tensor([[num_pages - 1], [num_pages - 7]], dtype=torch.int32, device="cuda")
  run(c.batch(k_pages=pool.data_ptr(), v_pages=values.data_ptr(), groups=2, num_pages=num_pages, tokens_per_page=page, max_pages_per_group=1, page_map=page_map.data_ptr()))
  for r, at in enumerate((num_pages - 1, num_pages - 7)):
    assert torch.equal(pool[0, at, int(c.pos[r])], c.k[r]) and torch.equal(values[0, at, int(c.pos[r])].cpu(), c.x[r, 256:])


def test_streams_and_graphs():
  c = Case(20, 4, 2, 64, 64, True, seed=6)
  side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
  torch.cuda.synchronize()
  with torch.cuda.graph(graph, stream=side):
    run(c.batch())
  for seed in range(3):
    c.pos = torch.randint(0, 5000, (20,), generator=torch.Generator().manual_seed(seed)).int()
    c.pos_dev.copy_(c.pos)
    graph.replay()
    q, k, _, qs, ks = c.want()
    assert close(c.q.cpu().view(20, 4, 64), q, qs, 1) and close(c.k.cpu().view(20, 2, 64), k, ks, 1)


def test_frequencies_of_the_library():
  lib, freq, amplitude = _lib.load(), (ctypes.c_double * 32)(), ctypes.c_float()
  _lib.check(lib.mtx_rotary_frequencies(64, 1e4, _lib.ROTARY["yarn"], 8.0, 2048.0, 1.0, 32.0, freq, ctypes.byref(amplitude)))
  c = Case(4, 2, 1, 64, 64, False, seed=5, amplitude=amplitude.value, most=16000)
  c.freq = torch.tensor(list(freq), dtype=torch.float64)
  c.freq_dev.copy_(c.freq)
  run(c.batch())
  q, k, _, qs, ks = c.want()
  assert close(c.q.cpu().view(4, 2, 64), q, qs, 1.3) and close(c.k.cpu().view(4, 1, 64), k, ks, 1.3)
