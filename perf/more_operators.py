"""What is measured of the operators that a step of drafted tokens needs around its products: requests that go on from one shared prompt (a voice, a
system text) and bring their last token and some drafted ones, a row each.

norm     the sum of the residual stream and a sublayer's output, its RMS norm, and the result in the next product's type: 8 bits with a scale per 128 values, or bfloat16
rotary   rotary positions for the projected queries and keys, and the keys and values into the pages of their sequences
attend   the rows' attention over the paged cache, where neighbouring sequences share the pages of a prefix
verify   the drafted tokens against the target's probabilities, with given random numbers: how many stay, and the token behind them

Widths, heads and vocabularies are those of the text-to-semantic GPT (1280 wide, 20 heads over 4 of 64 channels, 264,192 tokens), of the gemma3 models (2560 and 5376 wide, 8
heads over 4 of 256) and of the layered models of the benchmark (16 heads over 4 of 128, 16 over 8 of 64, 32,768 tokens).
"""

import math

import torch

own = False

BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
CODES = {"bf16": 0, "f32": 1, "fp8": 2}
EPS = 1e-5


def listed():
  return [
      # a decode step's rows in front of the fused query, key and value projection
      dict(name="norm decode 64", op="norm", rows=64, width=1280, x="bf16", residual="bf16", out="fp8"),
      # a portion of a prompt beside other requests' tokens, the residual stream in 32 bits
      dict(name="norm mixed 333", op="norm", rows=333, width=2560, x="bf16", residual="f32", out="bf16"),
      # a long prompt through a wide model
      dict(name="norm prompt 4096", op="norm", rows=4096, width=5376, x="bf16", residual="bf16", out="fp8"),
      # one request alone with its drafts
      dict(name="rotary drafts 5", op="rotary", sequences=1, tokens=5, heads=20, kv_heads=4, dim=64, rot=64, half=True, x="bf16", page=32, before=1200),
      # prompts of several requests in one step, half of every head rotated
      dict(name="rotary prompt 4001", op="rotary", sequences=3, tokens=4001, heads=16, kv_heads=4, dim=128, rot=64, half=False, x="bf16", page=64, before=90000),
      # two requests of a short preamble: launches and latency
      dict(name="attend pair", op="attend", sequences=2, drafts=0, prefixes=1, prefix=224, tail=40, heads=16, kv_heads=8, dim=64, page=16),
      # 64 utterances of one voice in the middle of their answers
      dict(name="attend tts 64", op="attend", sequences=64, drafts=0, prefixes=1, prefix=992, tail=1500, heads=20, kv_heads=4, dim=64, page=32),
      # two system texts, requests with up to four drafted tokens
      dict(name="attend drafts 48", op="attend", sequences=48, drafts=4, prefixes=2, prefix=4096, tail=700, heads=16, kv_heads=4, dim=128, page=64),
      # many short questions about one long document
      dict(name="attend document 128", op="attend", sequences=128, drafts=4, prefixes=1, prefix=16384, tail=512, heads=16, kv_heads=4, dim=128, page=64),
      # one request with a plain vocabulary
      dict(name="verify one", op="verify", sequences=1, drafts=4, vocab=32768, draft=True, greedy=False),
      # drafts that were looked up (no probabilities), some requests greedy
      dict(name="verify looked up 32", op="verify", sequences=32, drafts=3, vocab=32768, draft=False, greedy=True),
      # 64 utterances, every one with up to four drafted tokens of the expanded vocabulary
      dict(name="verify tts 64", op="verify", sequences=64, drafts=4, vocab=264192, draft=True, greedy=False),
  ]


def _log(rng, low, high):
  return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
  op = rng.choice(["norm", "norm", "rotary", "attend", "attend", "attend", "verify", "verify"])
  if op == "norm":
    width = _log(rng, 64, 21504)
    return dict(op=op, rows=_log(rng, 1, min(32768, 20_000_000 // width)), width=width, x=rng.choice(["bf16", "bf16", "f32"]), residual=rng.choice(["bf16", "bf16", "f32"]),
                out=rng.choice(["fp8", "fp8", "bf16", "f32"]))
  dim = rng.choice([64, 128, 128, 256])
  kv_heads = rng.choice([1, 2, 4, 8])
  heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
  if op == "rotary":
    tokens = _log(rng, 1, min(8192, 12_000_000 // (heads * dim)))
    return dict(op=op, sequences=_log(rng, 1, min(64, tokens)), tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, 2 * (dim // 5)]),
                half=rng.random() < 0.5, x=rng.choice(["bf16", "bf16", "f32"]), page=rng.choice([8, 16, 64]), before=_log(rng, 1, 100000))
  if op == "attend":
    sequences, drafts, tail, page = _log(rng, 1, 200), rng.choice([0, 0, 1, 4, 7]), _log(rng, 1, 3000), rng.choice([8, 16, 32, 64, 128])
    # no more keys than the largest listed case has per row, in all sequences together no more than fit when they are laid out one by one, and tails of 400 MB at most
    most = min(int(128 * 5 * 16 * 16896 * 128 / (sequences * (drafts + 1) * heads * dim)), int(128 * 16896 * 4 * 128 / (sequences * kv_heads * dim)))
    tail = max(1, min(tail, most // 3, 100_000_000 // (sequences * kv_heads * dim)))
    return dict(op=op, sequences=sequences, drafts=drafts, prefixes=min(sequences, rng.choice([1, 1, 2, 5])), prefix=_log(rng, 16, max(17, min(32768, most - tail))) // page * page,
                tail=tail, heads=heads, kv_heads=kv_heads, dim=dim, page=page)
  vocab, drafts = _log(rng, 1000, 264192), rng.choice([1, 2, 4, 7])
  return dict(op=op, sequences=_log(rng, 1, min(256, 64 * 5 * 264192 // (vocab * (drafts + 1)))), drafts=drafts, vocab=vocab, draft=rng.random() < 0.7, greedy=rng.random() < 0.3)


# ---- what a case's sizes say -----------------------------------------------------------------------------------------------------


def _spread(n, low, high):
  """n sizes between low and high, neighbours far apart, the last of them `high`."""
  return [low + (high - low) * ((7 * i + 7) % n + 1) // n if n % 7 else low + (high - low) * (i + 1) // n for i in range(n)]


def _rows_of(case):
  """Rows of each sequence: its last token and up to `drafts` drafted ones."""
  most = case["drafts"] + 1
  return [max(1, most - (i % 4 == 3) * (i % most)) for i in range(case["sequences"])]


def _tails(case):
  """Tokens of each sequence behind the prefix, its rows among them."""
  return [max(n, t) for n, t in zip(_rows_of(case), _spread(case["sequences"], (case["tail"] + 3) // 4, case["tail"]))]


def work(case):
  size = dict(bf16=2, f32=4, fp8=1)
  if case["op"] == "norm":
    n = case["rows"] * case["width"]
    return dict(bytes=n * (size[case["x"]] + 2 * size[case["residual"]] + size[case["out"]]) + case["width"] * 4 + (case["rows"] * -(-case["width"] // BLOCK) * 4 if case["out"] == "fp8" else 0),
                flops=5 * n)
  if case["op"] == "rotary":
    wide, tokens = (case["heads"] + 2 * case["kv_heads"]) * case["dim"], case["tokens"]
    return dict(bytes=tokens * (wide * (size[case["x"]] + 2) + 8), flops=tokens * (case["heads"] + case["kv_heads"]) * case["rot"] * 3)
  rows = sum(_rows_of(case))
  if case["op"] == "attend":
    tails, per_token = _tails(case), case["kv_heads"] * case["dim"] * 4
    return dict(bytes=(case["prefixes"] * case["prefix"] + sum(tails)) * per_token + rows * case["heads"] * case["dim"] * 4,
                flops=4 * case["heads"] * case["dim"] * sum(n * (case["prefix"] + t) for n, t in zip(_rows_of(case), tails)))
  read = rows + (rows - case["sequences"] if case["draft"] else 0)
  return dict(bytes=4 * read * case["vocab"], flops=4 * read * case["vocab"])


# ---- inputs ----------------------------------------------------------------------------------------------------------------------


def _generator(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def _ints(values):
  return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
  total, out = 0, [0]
  for n in counts:
    total += n
    out.append(total)
  return out


def _frequencies(dims, scaled):
  """Radians per position; scaled: the slow ones by a quarter, as for a context four times as long."""
  freq = 10000.0 ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
  return torch.where(freq < 2 * math.pi / 8192, freq / 4, freq) if scaled else freq


def prepare(case, seed):
  g = _generator(seed)
  if case["op"] == "norm":
    rows, width = case["rows"], case["width"]
    s = dict(case)
    s["x"] = torch.randn(rows, width, device="cuda", generator=g).to(TYPES[case["x"]])
    stream = 3 * torch.randn(rows, width, device="cuda", generator=g) * (1 + 15 * (torch.rand(width, device="cuda", generator=g) > 0.995))
    stream[rows // 2 + 1 :: 97] = 0  # rows of padding, with a sublayer's output or (some) without
    s["x"][rows // 2 + 1 :: 194] = 0
    s["residual"] = stream.to(TYPES[case["residual"]])
    s["weight"] = 1 + 0.3 * torch.randn(width, device="cuda", generator=g)
    s["sum"], s["scale"] = torch.empty_like(s["residual"]), None
    pitch = -(-width // 128) * 128
    s["out"] = torch.empty(rows, pitch, dtype=TYPES[case["out"]], device="cuda")
    if case["out"] == "fp8":
      s["scale"] = torch.empty(rows, pitch // BLOCK, device="cuda")
    s["types"] = [CODES[case[w]] for w in ("x", "residual", "out")]
    return s
  if case["op"] == "rotary":
    return _rotary_state(case, g)
  if case["op"] == "attend":
    return _attend_state(case, g)
  return _verify_state(case, g)


def _pages(counts, page, g, first=0):
  """Pages of each sequence, scattered over a pool; (the pool's pages, [sequences, most])."""
  total = sum(counts) + first
  order = torch.randperm(total, device="cuda", generator=g).int()
  most = max(counts)
  at = torch.tensor(_starts(counts)[:-1], device="cuda").view(-1, 1) + torch.arange(most, device="cuda").view(1, -1) + first
  return order, torch.where(torch.arange(most, device="cuda").view(1, -1) < torch.tensor(counts, device="cuda").view(-1, 1), order[at.clamp(max=total - 1)], 0)


def _rotary_state(case, g):
  sequences, tokens, page, wide = case["sequences"], case["tokens"], case["page"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
  n = [tokens // sequences + (i < tokens % sequences) for i in range(sequences)]
  # the pages of what came before are there, but a program that has forgotten the front of a sequence keeps pages for its end alone
  s = dict(case, projected=torch.randn(tokens, wide, device="cuda", generator=g).to(TYPES[case["x"]]))
  before = [case["before"] * (i + 1) // sequences for i in range(sequences)]
  used = [-(-(b + m) // page) - b // page for b, m in zip(before, n)]
  _, rows = _pages(used, page, g)
  most = max(b // page + u for b, u in zip(before, used))
  page_map = torch.zeros(sequences, most, dtype=torch.int32, device="cuda")
  for i in range(sequences):
    page_map[i, before[i] // page : before[i] // page + used[i]] = rows[i, : used[i]]
  s["page map"] = page_map
  s["group"] = _ints([i for i in range(sequences) for _ in range(n[i])])
  s["pos"] = _ints([before[i] + j for i in range(sequences) for j in range(n[i])])
  s["frequencies"] = _frequencies(case["rot"], case["before"] > 8192)
  s["amplitude"] = 1.0 if case["before"] <= 8192 else 1.1
  shape = (case["kv_heads"], sum(used), page, case["dim"])
  s["k pages"] = torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)
  s["v pages"] = torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)
  s["q"] = torch.empty(tokens, case["heads"] * case["dim"], dtype=torch.bfloat16, device="cuda")
  return s


def _attend_state(case, g):
  sequences, prefixes, page, dim = case["sequences"], case["prefixes"], case["page"], case["dim"]
  n, tails = _rows_of(case), _tails(case)
  shared = case["prefix"] // page  # whole pages
  used = [-(-t // page) for t in tails]
  order, rows = _pages(used, page, g, first=prefixes * shared)
  bounds = [sequences * i // prefixes for i in range(prefixes + 1)]
  of = torch.repeat_interleave(torch.arange(prefixes), torch.tensor([b - a for a, b in zip(bounds, bounds[1:])]))
  front = order[: prefixes * shared].view(prefixes, shared)[of.cuda()]
  s = dict(case, **{"page map": torch.cat([front, rows.int()], 1).contiguous(), "lengths": _ints([case["prefix"] + t for t in tails]), "row0": _ints(_starts(n)),
                    "prefix bounds": _ints(bounds), "prefix lengths": _ints([case["prefix"]] * prefixes), "rows": sum(n), "most rows": max(n)})
  shape = (case["kv_heads"], prefixes * shared + sum(used), page, dim)
  s["k pages"] = torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)
  s["v pages"] = torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)
  s["q"] = (2 * torch.randn(s["rows"], case["heads"] * dim, device="cuda", generator=g)).to(torch.bfloat16)
  s["out"] = torch.empty_like(s["q"])
  s["scale"] = dim**-0.5
  # what a program keeps for the call: the partial results of the pieces that an SM's share of the keys makes, a row of each head at a time
  s["scratch"] = torch.empty(_scratch_bytes(case, s["rows"]), dtype=torch.uint8, device="cuda")
  return s


def _scratch_bytes(case, rows):
  """An upper bound of mtx_prefix_attention_scratch_bytes: pieces of 128 rows of the prefixes' tiles, and of 16 rows of the tails'."""
  heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
  tiles = (rows * (heads // kv) // 64 + case["prefixes"] + 1) * kv + 2 * 148
  tails = (rows * (heads // kv) // 8 + case["sequences"] + 1) * kv + 8 * 148
  return (tiles * 128 + tails * 16) * (dim + 2) * 4 + (1 << 20)


def _verify_state(case, g):
  sequences, vocab = case["sequences"], case["vocab"]
  n = _rows_of(case)
  rows, row0 = sum(n), _starts(n)
  s = dict(case, row0=_ints(row0), rows=rows)
  target = 3 * torch.randn(rows, vocab, device="cuda", generator=g)
  of = torch.repeat_interleave(torch.arange(sequences), torch.tensor(n)).cuda()
  # two thirds of the requests may say tokens of the vocabulary's end alone, as utterances do
  target.masked_fill_((of % 3 != 2).view(-1, 1) & (torch.arange(vocab, device="cuda") < vocab - vocab // 4).view(1, -1), -math.inf)
  drafted = target + 0.7 * torch.randn(rows, vocab, device="cuda", generator=g)
  s["temperature"] = 0.6 + 0.8 * torch.rand(sequences, device="cuda", generator=g)
  if case["greedy"]:
    s["temperature"][::2] = 0
  # the draft's own draws; looked-up drafts are the likely token now and then
  noise = torch.empty(rows, vocab, device="cuda").exponential_(generator=g).log_()
  token = (drafted - noise).argmax(1)
  if not case["draft"]:
    token = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.6, target.argmax(1), token)
  s["token"] = torch.cat([token[:1], token[:-1]]).int()  # row r + 1 brings what was drafted at row r
  s["target"], s["drafted"] = target, drafted if case["draft"] else None
  s["accept"], s["pick"] = torch.rand(rows, device="cuda", generator=g), torch.rand(sequences, device="cuda", generator=g)
  s["accepted"], s["emitted"] = torch.empty(sequences, dtype=torch.int32, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
  s["scratch"] = torch.empty(rows * (vocab // 1024 + 2) * 64 + sequences * (vocab // 1024 + 2) * 32 + 65536, dtype=torch.uint8, device="cuda")
  return s


# ---- the operators ---------------------------------------------------------------------------------------------------------------


def run(state):
  s = state
  if own:
    return _own(s)
  if s["op"] == "norm":
    h = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
    v = h.float()
    y = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * s["weight"]
    if s["scale"] is None:
      return dict(sum=h, out=y.to(s["out"].dtype))
    rows, width = y.shape
    full = torch.nn.functional.pad(y, (0, s["out"].shape[1] - width)).view(rows, -1, BLOCK)
    largest = full.abs().amax(2).clamp(min=2.0**-96).double()
    q = (full * (448 / largest).float()[:, :, None]).to(torch.float8_e4m3fn).view(rows, -1)[:, :width]
    return dict(sum=h, out=q, scale=(largest / 448).float())
  if s["op"] == "rotary":
    return _plain_rotary(s)
  if s["op"] == "attend":
    return _plain_attend(s)
  return _plain_verify(s)


def _plain_rotary(s):
  heads, kv, dim, rot, page = s["heads"], s["kv_heads"], s["dim"], s["rot"], s["page"]
  tokens = s["tokens"]
  x = s["projected"].float().view(tokens, heads + 2 * kv, dim)
  angle = s["pos"].double()[:, None] * s["frequencies"]
  cos, sin = (torch.cos(angle) * s["amplitude"]).float()[:, None], (torch.sin(angle) * s["amplitude"]).float()[:, None]
  turned = x[:, : heads + kv, :rot]
  if s["half"]:
    a, b = turned[..., : rot // 2], turned[..., rot // 2 :]
    turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
  else:
    a, b = turned[..., 0::2], turned[..., 1::2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
  y = torch.cat([turned, x[:, : heads + kv, rot:]], -1).to(torch.bfloat16)
  at, slot = s["page map"][s["group"].long(), s["pos"].long() // page].long(), s["pos"].long() % page
  s["k pages"][:, at, slot] = y[:, heads:].transpose(0, 1)
  s["v pages"][:, at, slot] = x[:, heads + kv :].to(torch.bfloat16).transpose(0, 1)
  return dict(q=y[:, :heads].reshape(tokens, -1), k=s["k pages"], v=s["v pages"])


def _plain_attend(s):
  kv, dim, page, sequences, most = s["kv_heads"], s["dim"], s["page"], s["sequences"], s["most rows"]
  group = s["heads"] // kv
  row0, lengths = s["row0"].long(), s["lengths"].long()
  n = row0[1:] - row0[:-1]
  row = row0[:-1, None] + torch.arange(most, device="cuda")
  there = torch.arange(most, device="cuda") < n[:, None]
  q = s["q"].float()[row.clamp(max=s["rows"] - 1)].view(sequences, most, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(sequences, kv, most * group, dim)
  maps = s["page map"].long()
  keys = s["k pages"][:, maps].float().view(kv, sequences, -1, dim).transpose(0, 1)
  scores = (q @ keys.transpose(2, 3) * s["scale"]).view(sequences, kv, most, group, -1)
  del keys
  seen = (lengths - n)[:, None] + torch.arange(1, most + 1, device="cuda")
  mask = torch.arange(scores.shape[-1], device="cuda") < seen[:, :, None]
  scores = torch.where(mask[:, None, :, None], scores, -math.inf)
  p = torch.exp(scores - scores.amax(-1, keepdim=True))
  p = p / p.sum(-1, keepdim=True)
  values = s["v pages"][:, maps].float().view(kv, sequences, -1, dim).transpose(0, 1)
  out = (p.view(sequences, kv, most * group, -1) @ values).view(sequences, kv, most, group, dim).permute(0, 2, 1, 3, 4).reshape(sequences, most, -1)
  return out[there].to(torch.bfloat16)


def _first_largest(x):
  return torch.where(x == x.amax(1, keepdim=True), torch.arange(x.shape[1], device=x.device), x.shape[1]).amin(1)


def _plain_verify(s):
  """In 64 bits: a drawn number lies next to the border of two tokens, and a sum runs over all of them."""
  sequences, rows, vocab = s["sequences"], s["rows"], s["vocab"]
  row0 = s["row0"].long()
  of = torch.repeat_interleave(torch.arange(sequences, device="cuda"), row0[1:] - row0[:-1], output_size=rows)
  greedy = s["temperature"] == 0
  heat = torch.where(greedy, 1.0, s["temperature"]).double()[of, None]
  best = _first_largest(s["target"])

  def probabilities(logits):
    l = logits.double() / heat
    e = torch.exp(l - l.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)

  p = probabilities(s["target"])
  index = torch.arange(rows, device="cuda")
  last = index == row0[1:][of] - 1
  token = torch.roll(s["token"].long(), -1)  # what row r's logits decide on
  if s["drafted"] is None:
    q_of = torch.ones(rows, dtype=torch.float64, device="cuda")
  else:
    q = probabilities(s["drafted"])
    q_of = q[index, token]
  stays = torch.where(greedy[of], token == best, s["accept"].double() * q_of < p[index, token]) & ~last
  stop = torch.full((sequences,), rows, device="cuda").scatter_reduce_(0, of, torch.where(stays, rows, index), "amin")
  left = p[stop]
  if s["drafted"] is None:
    left[torch.arange(sequences, device="cuda"), token[stop]] *= last[stop]
  else:
    left = (left - q[stop] * ~last[stop][:, None]).clamp(min=0)
  left = torch.where(left.sum(1, keepdim=True) > 0, left, p[stop])
  up = left.cumsum(1)
  drawn = (up <= s["pick"].double()[:, None] * up[:, -1:]).sum(1)
  drawn = torch.minimum(drawn, torch.where(left > 0, torch.arange(vocab, device="cuda"), 0).amax(1))
  drawn = torch.where(greedy, best[stop], drawn)
  emitted = torch.where(index < stop[of], token, torch.where(index == stop[of], drawn[of], -1))
  return dict(accepted=(stop - row0[:-1]).int(), emitted=emitted.int())


def _ptr(t):
  return 0 if t is None else t.data_ptr()


def _own(s):
  from maxtext_indextts2_b200 import _lib

  lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
  if s["op"] == "norm":
    x, r, h, out, (x_type, r_type, o_type) = s["x"], s["residual"], s["sum"], s["out"], s["types"]
    _lib.check(lib.mtx_add_rmsnorm(x.data_ptr(), x_type, x.stride(0), r.data_ptr(), r_type, r.stride(0), h.data_ptr(), h.stride(0), s["weight"].data_ptr(), _lib.F32, 0.0, EPS,
                                   out.data_ptr(), o_type, out.stride(0), _ptr(s["scale"]), s["rows"], s["width"], stream))
    return dict(sum=h, out=out[:, : s["width"]]) if s["scale"] is None else dict(sum=h, out=out[:, : s["width"]], scale=s["scale"])
  if s["op"] == "rotary":
    x, q, wide = s["projected"], s["q"], s["heads"] * s["dim"]
    size, ld = x.element_size(), x.stride(0)
    kv_wide = s["kv_heads"] * s["dim"]
    batch = _lib.RotaryBatch(
        rows=s["tokens"], heads=s["heads"], kv_heads=s["kv_heads"], dim=s["dim"], rot_dims=s["rot"], rot_half=int(s["half"]), amplitude=s["amplitude"], freq=s["frequencies"].data_ptr(),
        pos=s["pos"].data_ptr(), type=CODES[s["x"]], q=x.data_ptr(), ldq=ld, k=x.data_ptr() + wide * size, ldk=ld, v=x.data_ptr() + (wide + kv_wide) * size, ldv=ld, out_type=_lib.BF16,
        q_out=q.data_ptr(), ldq_out=q.stride(0), k_pages=s["k pages"].data_ptr(), v_pages=s["v pages"].data_ptr(), groups=s["sequences"], num_pages=s["k pages"].shape[1],
        tokens_per_page=s["page"], max_pages_per_group=s["page map"].shape[1], group=s["group"].data_ptr(), page_map=s["page map"].data_ptr())
    _lib.check(lib.mtx_rotary(batch, stream))
    return dict(q=q, k=s["k pages"], v=s["v pages"])
  if s["op"] == "attend":
    q, out, k = s["q"], s["out"], s["k pages"]
    batch = _lib.PrefixBatch(rows=s["rows"], sequences=s["sequences"], row0=s["row0"].data_ptr(), lengths=s["lengths"].data_ptr(), page_map=s["page map"].data_ptr(),
                             prefixes=s["prefixes"], prefix_seq0=s["prefix bounds"].data_ptr(), prefix_len=s["prefix lengths"].data_ptr())
    _lib.check(lib.mtx_prefix_attention(q.data_ptr(), q.stride(0), k.data_ptr(), s["v pages"].data_ptr(), batch, out.data_ptr(), out.stride(0), s["heads"], s["kv_heads"], s["dim"],
                                        k.shape[1], s["page"], s["page map"].shape[1], s["scale"], 0.0, s["scratch"].data_ptr(), s["scratch"].numel(), stream))
    return out
  batch = _lib.DraftBatch(rows=s["rows"], sequences=s["sequences"], vocab=s["vocab"], row0=s["row0"].data_ptr(), token=s["token"].data_ptr(), target=s["target"].data_ptr(),
                          ld_target=s["target"].stride(0), draft=_ptr(s["drafted"]), ld_draft=0 if s["drafted"] is None else s["drafted"].stride(0),
                          temperature=s["temperature"].data_ptr(), accept_u=s["accept"].data_ptr(), pick_u=s["pick"].data_ptr())
  _lib.check(lib.mtx_verify_drafts(batch, s["accepted"].data_ptr(), s["emitted"].data_ptr(), s["scratch"].data_ptr(), s["scratch"].numel(), stream))
  return dict(accepted=s["accepted"], emitted=s["emitted"])


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def _e4m3(v):
  """The nearest value with four significant bits, exponents from -6 to 8, at most 448 in size; ties to the even one."""
  size = v.abs()
  _, e = torch.frexp(size)
  step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
  return torch.sign(v) * torch.minimum(torch.round(size / step) * step, torch.full_like(size, 448))


def exact(case, seed):
  s = prepare(case, seed)
  return dict(norm=_exact_norm, rotary=_exact_rotary, attend=_exact_attend, verify=_exact_verify)[case["op"]](s)


def _exact_norm(s):
  # the stored sum is rounded to its type by definition, the scales' fractions to 32 bits
  h = (s["x"].double() + s["residual"].double()).float().to(s["residual"].dtype).double()
  y = h / torch.sqrt(h.square().sum(1) / s["width"] + EPS)[:, None] * s["weight"].double()
  if s["scale"] is None:
    return dict(sum=h, out=y)
  scales, q = [], torch.empty_like(y)
  for c in range(0, s["width"], BLOCK):
    part = y[:, c : c + BLOCK]
    largest = part.abs().max(1).values.clamp(min=2.0**-96)
    scales.append((largest / 448).float().double())
    q[:, c : c + BLOCK] = _e4m3(part * (448 / largest).float().double()[:, None])
  return dict(sum=h, out=q, scale=torch.stack(scales, 1))


def _exact_rotary(s):
  heads, kv, dim, rot = s["heads"], s["kv_heads"], s["dim"], s["rot"]
  x = s["projected"].double()
  pair = torch.arange(rot // 2, device="cuda")
  first, second = (pair, pair + rot // 2) if s["half"] else (2 * pair, 2 * pair + 1)
  turn = torch.polar(torch.full((s["tokens"], rot // 2), s["amplitude"], dtype=torch.float64, device="cuda"), s["pos"].double()[:, None] * s["frequencies"])
  for h in range(heads + kv):
    z = torch.complex(x[:, h * dim + first], x[:, h * dim + second]) * turn
    x[:, h * dim + first], x[:, h * dim + second] = z.real, z.imag
  k, v = s["k pages"].double(), s["v pages"].double()
  page = s["page"]
  where = s["page map"].long().gather(1, torch.arange(s["page map"].shape[1], device="cuda").expand(s["sequences"], -1))
  slot = where[s["group"].long(), s["pos"].long().div(page, rounding_mode="floor")] * page + s["pos"].long() % page
  for h in range(kv):
    k[h].view(-1, dim).index_copy_(0, slot, x[:, (heads + h) * dim : (heads + h + 1) * dim])
    v[h].view(-1, dim).index_copy_(0, slot, x[:, (heads + kv + h) * dim : (heads + kv + h + 1) * dim])
  return dict(q=x[:, : heads * dim], k=k, v=v)


def _exact_attend(s):
  if s["rows"] * s["heads"] * int(s["lengths"].max()) * s["dim"] > 3e10:
    return None  # (minutes)
  heads, kv, dim = s["heads"], s["kv_heads"], s["dim"]
  out = torch.empty(s["rows"], heads * dim, dtype=torch.float64, device="cuda")
  row0, lengths = s["row0"].tolist(), s["lengths"].tolist()
  for i in range(s["sequences"]):
    n, size = row0[i + 1] - row0[i], lengths[i]
    pages = s["page map"][i, : -(-size // s["page"])].long()
    hidden = torch.triu(torch.ones(n, size, dtype=torch.bool, device="cuda"), size - n + 1)
    for h in range(kv):
      k = s["k pages"][h, pages].reshape(-1, dim)[:size].double()
      v = s["v pages"][h, pages].reshape(-1, dim)[:size].double()
      for a in range(h * (heads // kv), (h + 1) * (heads // kv)):
        weights = torch.softmax((s["q"][row0[i] : row0[i + 1], a * dim : (a + 1) * dim].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf), 1)
        out[row0[i] : row0[i + 1], a * dim : (a + 1) * dim] = weights @ v
  return out


def _exact_verify(s):
  row0, token = s["row0"].tolist(), s["token"].tolist()
  accepted, emitted = [], [-1] * s["rows"]
  for i in range(s["sequences"]):
    heat, kept, drawn = float(s["temperature"][i]), 0, None
    for r in range(row0[i], row0[i + 1]):
      final = r + 1 == row0[i + 1]
      l = s["target"][r].double()
      if heat == 0:
        best = int((l == l.max()).nonzero()[0, 0])
        keep, left = not final and token[r + 1] == best, None
      else:
        left = torch.softmax(l / heat, 0)
        keep = False
        if not final:
          x = token[r + 1]
          q = None if s["drafted"] is None else torch.softmax(s["drafted"][r].double() / heat, 0)
          keep = float(s["accept"][r]) * (1.0 if q is None else float(q[x])) < float(left[x])
          if not keep and q is not None:
            left = torch.relu(left - q)
          elif not keep:
            left[x] = 0
      if keep:
        emitted[r] = token[r + 1]
        kept += 1
        continue
      if left is None:
        drawn = best
      else:
        up = torch.cumsum(left, 0)
        drawn = min(int(torch.searchsorted(up, up[-1] * float(s["pick"][i]), right=True)), int(left.nonzero()[-1, 0]))
      emitted[r] = drawn
      break
    accepted.append(kept)
  return dict(accepted=_ints(accepted), emitted=_ints(emitted))
