"""Steps of drafted tokens as a server runs them: requests of one voice go on from a shared prompt; norm, 8-bit products, rotary positions, attention, verification and the
record of emitted tokens follow one another on one stream.  Every operator is held against its definition in 64 bits on what the one in front of it left."""

import ctypes

import pytest
import torch

from maxtext_indextts2_b200 import _lib
from tests import draft_helpers as ref
from tests import fp8_helpers

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


class Server:
  """One layer: x -> norm -> q, k, v -> rotary, pages -> attention -> projection -> sum, norm -> vocabulary -> verification -> record."""

  def __init__(self, sequences, drafts, prefix, width=256, heads=6, kv=2, dim=64, vocab=777, page=16, room=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    self.lib, self.sequences, self.n, self.rows, self.prefix = _lib.load(), sequences, drafts + 1, sequences * (drafts + 1), prefix
    self.width, self.heads, self.kv, self.dim, self.vocab, self.page = width, heads, kv, dim, vocab, page
    self.wide = (heads + 2 * kv) * dim
    self.embedding = torch.randn(vocab, width, generator=g).to(BF16).cuda()
    self.weights = {}
    for name, n, k in (("qkv", self.wide, width), ("wo", width, heads * dim), ("head", vocab, width)):
      w = (torch.randn(n, k, generator=g) * (3 if name == "qkv" else 1) * k**-0.5).to(BF16).cuda()
      q, s = torch.empty(n, fp8_helpers.pitch(k), dtype=torch.uint8, device="cuda"), torch.empty(-(-n // 128), -(-k // 128), device="cuda")
      _lib.check(self.lib.mtx_quantize_fp8(w.data_ptr(), _lib.BF16, k, n, k, 128, q.data_ptr(), q.stride(0), s.data_ptr(), self.stream()))
      self.weights[name] = (q, s, n, k)
    self.norms = [(1 + 0.2 * torch.randn(width, generator=g)).cuda() for _ in range(2)]
    freq, amplitude = (ctypes.c_double * (dim // 2))(), ctypes.c_float()
    _lib.check(self.lib.mtx_rotary_frequencies(dim, 1e4, _lib.ROTARY["bands"], 4.0, 512.0, 1.0, 4.0, freq, ctypes.byref(amplitude)))
    self.freq, self.amplitude = torch.tensor(list(freq), dtype=torch.float64).cuda(), amplitude.value
    shared, own = prefix // page, 6
    self.num_pages = shared + own * sequences
    order = torch.randperm(self.num_pages, generator=g).int()
    self.page_map = torch.cat([order[:shared].expand(sequences, -1), order[shared:].view(sequences, own), torch.zeros(sequences, room, dtype=torch.int32)], 1).contiguous().cuda()
    self.k = torch.randn(kv, self.num_pages, page, dim, generator=g).to(BF16).cuda()
    self.v = torch.randn(kv, self.num_pages, page, dim, generator=g).to(BF16).cuda()
    e = lambda *shape, t=BF16: torch.empty(*shape, dtype=t, device="cuda")
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    self.x, self.h = e(self.rows, width), e(self.rows, width)
    self.row0, self.bounds, self.prefix_len = i([self.n * s for s in range(sequences + 1)]), i([0, sequences]), i([prefix])
    self.group, self.slot = i([s for s in range(sequences) for _ in range(self.n)]), i([s for s in range(sequences) for _ in range(self.n)])
    self.token, self.pos, self.lengths = i([0] * self.rows), i([0] * self.rows), i([0] * sequences)
    self.normed, self.normed_scale = e(self.rows, width, t=FP8), e(self.rows, width // 128, t=torch.float32)
    self.projected, self.q, self.attended = e(self.rows, self.wide), e(self.rows, heads * dim), e(self.rows, heads * dim)
    self.sub, self.second, self.second_scale = e(self.rows, width), e(self.rows, width, t=FP8), e(self.rows, width // 128, t=torch.float32)
    self.logits, self.drafted = e(self.rows, vocab, t=torch.float32), e(self.rows, vocab, t=torch.float32)
    self.temperature = torch.tensor([0.0, 0.9, 1.2, 0.7] * sequences)[:sequences].cuda()
    self.accept, self.pick = e(self.rows, t=torch.float32), e(sequences, t=torch.float32)
    self.accepted, self.emitted = i([0] * sequences), i([0] * self.rows)
    self.seen, self.touched = torch.zeros(sequences, -(-vocab // 8) * 8, dtype=torch.int16, device="cuda"), torch.zeros(sequences, -(-vocab // 256), dtype=torch.int32, device="cuda")
    bytes_ = lambda n: torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    self.product_scratch = bytes_(self.lib.mtx_linear_fp8_scratch_bytes(self.rows, heads * dim))
    self.attention_scratch = bytes_(self.lib.mtx_prefix_attention_scratch_bytes(self.rows, sequences, 1, heads, kv, dim))
    self.verify_scratch = bytes_(self.lib.mtx_verify_drafts_scratch_bytes(self.rows, sequences, vocab))
    self.length = [prefix + 3 + 2 * s for s in range(sequences)]  # tokens in the pages before the step
    self.gen = g

  def stream(self):
    return torch.cuda.current_stream().cuda_stream

  def linear(self, x, scale, name, out):
    q, s, n, k = self.weights[name]
    fp8 = x.dtype == FP8
    _lib.check(self.lib.mtx_linear_fp8(x.data_ptr(), _lib.E4M3 if fp8 else _lib.BF16, x.stride(0), scale.data_ptr() if fp8 else None, q.data_ptr(), q.stride(0), s.data_ptr(), out.data_ptr(),
                                       _lib.F32 if out.dtype == torch.float32 else _lib.BF16, n, self.rows, n, k, self.product_scratch.data_ptr(), self.product_scratch.numel(), self.stream()))

  def norm(self, x, residual, total, weight, out, scale):
    _lib.check(self.lib.mtx_add_rmsnorm(x.data_ptr(), _lib.BF16, self.width, None if residual is None else residual.data_ptr(), _lib.BF16, self.width, None if total is None else total.data_ptr(),
                                        self.width, weight.data_ptr(), _lib.F32, 0.0, 1e-5, out.data_ptr(), _lib.E4M3, self.width, scale.data_ptr(), self.rows, self.width, self.stream()))

  def step(self):
    lib = self.lib
    self.norm(self.x, None, None, self.norms[0], self.normed, self.normed_scale)
    self.linear(self.normed, self.normed_scale, "qkv", self.projected)
    at, d = self.projected.data_ptr(), 2 * self.dim
    _lib.check(lib.mtx_rotary(_lib.RotaryBatch(
        rows=self.rows, heads=self.heads, kv_heads=self.kv, dim=self.dim, rot_dims=self.dim, rot_half=1, amplitude=self.amplitude, type=_lib.BF16, out_type=_lib.BF16,
        freq=self.freq.data_ptr(), pos=self.pos.data_ptr(), q=at, ldq=self.wide, k=at + self.heads * d, ldk=self.wide, v=at + (self.heads + self.kv) * d, ldv=self.wide, q_out=self.q.data_ptr(),
        ldq_out=self.heads * self.dim, k_pages=self.k.data_ptr(), v_pages=self.v.data_ptr(), groups=self.sequences, num_pages=self.num_pages, tokens_per_page=self.page,
        max_pages_per_group=self.page_map.shape[1], group=self.group.data_ptr(), page_map=self.page_map.data_ptr()), self.stream()))
    batch = _lib.PrefixBatch(rows=self.rows, sequences=self.sequences, row0=self.row0.data_ptr(), lengths=self.lengths.data_ptr(), page_map=self.page_map.data_ptr(), prefixes=1,
                             prefix_seq0=self.bounds.data_ptr(), prefix_len=self.prefix_len.data_ptr())
    _lib.check(lib.mtx_prefix_attention(self.q.data_ptr(), self.heads * self.dim, self.k.data_ptr(), self.v.data_ptr(), batch, self.attended.data_ptr(), self.heads * self.dim, self.heads, self.kv,
                                        self.dim, self.num_pages, self.page, self.page_map.shape[1], self.dim**-0.5, 0.0, self.attention_scratch.data_ptr(), self.attention_scratch.numel(),
                                        self.stream()))
    self.linear(self.attended, None, "wo", self.sub)
    self.norm(self.sub, self.x, self.h, self.norms[1], self.second, self.second_scale)
    self.linear(self.second, self.second_scale, "head", self.logits)
    drafts = _lib.DraftBatch(rows=self.rows, sequences=self.sequences, vocab=self.vocab, row0=self.row0.data_ptr(), token=self.token.data_ptr(), target=self.logits.data_ptr(), ld_target=self.vocab,
                             draft=self.drafted.data_ptr(), ld_draft=self.vocab, temperature=self.temperature.data_ptr(), accept_u=self.accept.data_ptr(), pick_u=self.pick.data_ptr())
    _lib.check(lib.mtx_verify_drafts(drafts, self.accepted.data_ptr(), self.emitted.data_ptr(), self.verify_scratch.data_ptr(), self.verify_scratch.numel(), self.stream()))
    _lib.check(lib.mtx_note_tokens(self.seen.data_ptr(), self.seen.stride(0), self.touched.data_ptr(), self.touched.stride(0), self.sequences, self.vocab, self.emitted.data_ptr(),
                                   self.slot.data_ptr(), self.rows, 0, self.stream()))

  def new_inputs(self, last, drafts):
    """last [sequences], drafts [sequences, n - 1]: the step's tokens; their positions and what the draft said come along."""
    token = torch.cat([last[:, None], drafts], 1).int().reshape(-1)
    self.token.copy_(token)
    self.x.copy_(self.embedding[token.long().cuda()])
    self.lengths.copy_(torch.tensor([l + self.n for l in self.length], dtype=torch.int32))
    self.pos.copy_(torch.tensor([l + i for l in self.length for i in range(self.n)], dtype=torch.int32))
    self.drafted.copy_(2 * torch.randn(self.rows, self.vocab, generator=self.gen))
    self.accept.copy_(torch.rand(self.rows, generator=self.gen))
    self.pick.copy_(torch.rand(self.sequences, generator=self.gen))

  def dequantised(self, q, s, rows, block):
    k = q.shape[1]
    return q.view(FP8).double()[:rows] * s.double().repeat_interleave(block, 0)[:rows].repeat_interleave(128, 1)[:, :k]

  def product(self, x, scale, name, out):
    q, s, n, k = self.weights[name]
    if x.dtype == FP8:
      a = self.dequantised(x, scale, self.rows, 1)
    else:
      v, sc = fp8_helpers.quantised(x.cpu(), 1)
      a = (v * fp8_helpers.spread(sc, 1, self.rows, k)).cuda()
    w = self.dequantised(q, s, n, 128)[:, :k]
    want, size = a @ w.T, a.abs() @ w.abs().T
    half = ref.EPS[out.dtype]
    assert bool(((out.double() - want).abs() <= size * (132 * 2.0**-23 + 12 * 2.0**-24) * (1 + half) + half * want.abs()).all())

  def check(self, k_before, v_before, seen_before):
    """The step that has run, operator by operator."""
    f = lambda t: t.double().cpu()
    _, y = ref.normed(self.x, None, self.norms[0], 0.0, 1e-5, None)
    ref.eight_bits(f(y), f(self.normed), f(self.normed_scale))
    self.product(self.normed, self.normed_scale, "qkv", self.projected)
    x = self.projected.cpu().view(self.rows, -1, self.dim)
    turned = ref.rotated(x[:, : self.heads + self.kv], self.pos.cpu(), self.freq.cpu(), self.amplitude, True)
    size = 2 * x.double().abs().amax(2, keepdim=True)[:, : self.heads + self.kv]
    got = torch.cat([self.q.cpu().view(self.rows, self.heads, self.dim), torch.empty(self.rows, self.kv, self.dim, dtype=BF16)], 1)
    k_want, v_want = k_before.clone(), v_before.clone()
    for r in range(self.rows):
      s, p = int(self.group[r]), int(self.pos[r])
      page = int(self.page_map[s, p // self.page])
      got[r, self.heads :] = self.k[:, page, p % self.page].cpu()
      k_want[:, page, p % self.page], v_want[:, page, p % self.page] = self.k[:, page, p % self.page], self.projected[r].view(-1, self.dim)[self.heads + self.kv :]
    assert bool(((got.double() - turned).abs() <= 2.0**-20 * self.amplitude * size + 2.0**-8 * (turned.abs() + 2.0**-20 * size)).all())
    assert torch.equal(self.k, k_want) and torch.equal(self.v, v_want)
    want, bound = ref.attention(self.q, self.k, self.v, self.row0.tolist(), self.lengths.tolist(), self.page_map, self.heads, self.dim**-0.5)
    assert bool(((self.attended.double().view_as(want) - want).abs() <= bound).all())
    self.product(self.attended, None, "wo", self.sub)
    h, y = ref.normed(self.sub.cpu(), self.x.cpu(), self.norms[1].cpu(), 0.0, 1e-5, BF16)
    assert torch.equal(f(self.h), h)
    ref.eight_bits(y, f(self.second), f(self.second_scale))
    self.product(self.second, self.second_scale, "head", self.logits)
    heat = f(self.temperature)
    for s, (kept, tokens, near, (low, high)) in enumerate(ref.verified(self.logits.cpu(), self.drafted.cpu(), self.row0.tolist(), self.token.cpu(), heat, heat, f(self.accept), f(self.pick), self.vocab)):
      got = self.emitted[s * self.n : (s + 1) * self.n].tolist()
      assert not near and int(self.accepted[s]) == kept and got[:kept] == tokens[:kept] and low <= got[kept] <= high and got[kept + 1 :] == tokens[kept + 1 :]
    words = seen_before.cpu().int()
    for s in range(self.sequences):
      for t in self.emitted[s * self.n : (s + 1) * self.n].tolist():
        if t >= 0:
          words[s, t] += 1
    assert torch.equal(self.seen.cpu().int(), words)


@pytest.mark.parametrize("sequences,drafts,prefix,room", [(1, 0, 0, 0), (1, 3, 64, 0), (9, 2, 160, 0), (40, 3, 96, 0), (40, 3, 96, 600)])  # (with room for 9600 tokens more: on the tensor cores)
@pytest.mark.parametrize("captured", [False, True])
def test_steps(sequences, drafts, prefix, room, captured):
  s = Server(sequences, drafts, prefix, room=room, seed=sequences)
  if captured:
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    for t in (s.x, s.drafted, s.accept, s.pick):
      t.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
      s.step()
  last = torch.randint(0, s.vocab, (sequences,), generator=s.gen)
  kept = 0
  for step in range(4):
    guess = torch.randint(0, s.vocab, (sequences, drafts), generator=s.gen)
    s.new_inputs(last, guess)
    if drafts and step:  # greedy requests whose drafts are what the model says: found by running the step once for its logits
      seen, touched, k, v = s.seen.clone(), s.touched.clone(), s.k.clone(), s.v.clone()
      s.step()
      best = s.logits.view(sequences, s.n, s.vocab).argmax(2).cpu()
      guess[:, 0] = best[:, 0]
      accept, pick = s.accept.clone(), s.pick.clone()
      s.new_inputs(last, guess)
      for a, b in ((s.seen, seen), (s.touched, touched), (s.k, k), (s.v, v), (s.accept, accept), (s.pick, pick)):
        a.copy_(b)
    k, v, seen = s.k.clone(), s.v.clone(), s.seen.clone()
    graph.replay() if captured else s.step()
    s.check(k, v, seen)
    for i in range(sequences):  # what was emitted is the sequence's; the drafts that did not stay are overwritten by the next step
      n = int(s.accepted[i])
      kept += n
      s.length[i] += n + 1
      last[i] = int(s.emitted[i * s.n + n])
  assert kept > 0 or drafts == 0
