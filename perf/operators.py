"""What is measured of the operators around the answering end of a step: products with 8-bit weights, and the controls of the logits that such a
product over the vocabulary gives.

quantize  float8_e4m3fn values with one scale per 128 values of a row (activations) or per 128 x 128 block (weights)
linear    x W^T with W in that form; x comes as bfloat16 or float32 (then it is quantised within the call), or quantised already
control   penalties for tokens that a request has seen, biases and masks of allowed tokens, on a batch's logits
note      the record of seen tokens that the penalties read: the prompts' tokens, then one token per request and step

Widths, hidden sizes and vocabularies are those of the text-to-semantic GPT (1280, 5120, 264,192 tokens), of the gemma3 models (2560 and 5376 wide)
and of the layered models of the benchmark (2048 wide, 32,768 tokens).  Weights are random with the spread of trained ones, activations random
with a few channels that stand out, as they do behind a norm.
"""

import math

import torch

own = False

BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}
CODES = {"bf16": 0, "f32": 1, "fp8": 2}


def listed():
  return [
      # a decode step's activations: one row per request
      dict(name="quantize decode 64", op="quantize", rows=64, k=1280, block=1, type="bf16"),
      # a long prompt's hidden activations in front of the down-projection
      dict(name="quantize prompt 4001", op="quantize", rows=4001, k=10240, block=1, type="bf16"),
      # loading a model: the vocabulary projection of the text-to-semantic GPT
      dict(name="quantize head", op="quantize", rows=264192, k=1280, block=128, type="bf16"),
      # one request alone: the fused query, key and value projection; launches and latency
      dict(name="linear token", op="linear", rows=1, k=1280, n=1792, x="bf16", out="bf16"),
      # the down-projection of a decode step: few columns, a long sum
      dict(name="linear decode 64", op="linear", rows=64, k=5120, n=1280, x="bf16", out="bf16"),
      # the expanded vocabulary of a decode step, the largest weight there is
      dict(name="linear head 64", op="linear", rows=64, k=1280, n=264192, x="bf16", out="f32"),
      # a portion of a prompt beside other requests' tokens
      dict(name="linear mixed 333", op="linear", rows=333, k=2560, n=10240, x="bf16", out="bf16"),
      # a long prompt through a wide model, activations quantised by the operator before
      dict(name="linear prompt 4096", op="linear", rows=4096, k=5376, n=21504, x="fp8", out="bf16"),
      # one request with a plain vocabulary
      dict(name="control one", op="control", rows=1, vocab=32000, history=300, masks=1, biases=16),
      # 64 utterances at once: most rows may only say audio tokens, a few are free, one has nothing left to say
      dict(name="control tts 64", op="control", rows=64, vocab=264192, history=1500, masks=3, biases=40),
      # every request's new token
      dict(name="note step 64", op="note", slots=64, vocab=264192, tokens=64, prompt=False),
      # the prompts of a full batch
      dict(name="note prompts", op="note", slots=64, vocab=264192, tokens=61234, prompt=True),
  ]


def _log(rng, low, high):
  return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
  op = rng.choice(["quantize", "linear", "linear", "linear", "control", "control", "note"])
  if op == "quantize":
    block = rng.choice([1, 1, 128])
    k = _log(rng, 16, 21504)
    return dict(op=op, rows=_log(rng, 1, min(65536, 300_000_000 // k)), k=k, block=block, type=rng.choice(["bf16", "bf16", "f32"]))
  if op == "linear":
    k = _log(rng, 64, 21504)
    n = _log(rng, 16, min(264192, 330_000_000 // k))
    rows = _log(rng, 1, max(1, min(8192, int(0.9 * 4096 * 5376 * 21504 / (n * k)), 200_000_000 // n)))
    return dict(op=op, rows=rows, k=k, n=n, x=rng.choice(["bf16", "bf16", "f32", "fp8"]), out=rng.choice(["bf16", "f32"]))
  if op == "control":
    vocab = _log(rng, 1000, 264192)
    return dict(op=op, rows=_log(rng, 1, min(256, 64 * 264192 // vocab)), vocab=vocab, history=_log(rng, 1, 8000), masks=rng.choice([0, 1, 5]), biases=rng.choice([0, 3, 300]))
  slots = _log(rng, 1, 256)
  return dict(op=op, slots=slots, vocab=_log(rng, 1000, min(264192, 64 * 264192 // slots)), tokens=_log(rng, slots, 65536), prompt=rng.random() < 0.5)


def work(case):
  if case["op"] == "quantize":
    rows, k, size = case["rows"], case["k"], 4 if case["type"] == "f32" else 2
    return dict(bytes=rows * k * (size + 1) + -(-rows // case["block"]) * -(-k // BLOCK) * 4, flops=2 * rows * k)
  if case["op"] == "linear":
    rows, k, n, blocks = case["rows"], case["k"], case["n"], -(-case["k"] // BLOCK)
    x = rows * k * dict(bf16=2, f32=4, fp8=1)[case["x"]] + (rows * blocks * 4 if case["x"] == "fp8" else 0)
    return dict(bytes=x + n * k + -(-n // BLOCK) * blocks * 4 + rows * n * (4 if case["out"] == "f32" else 2), flops=2 * rows * k * n)
  if case["op"] == "control":
    rows, vocab = case["rows"], case["vocab"]
    return dict(bytes=rows * vocab * 8 + case["masks"] * -(-vocab // 8) + rows * (case["history"] * 2 + case["biases"] * 8), flops=2 * rows * vocab)
  return dict(bytes=case["tokens"] * (4 + 4 + 2 + 2), flops=case["tokens"])


# ---- inputs ---------------------------------------------------------------------------------------------------------------------


def _generator(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, k, g):
  x = torch.randn(rows, k, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
  x *= 1 + 20 * (torch.rand(k, device="cuda", generator=g) > 0.995)
  x[rows // 2 + 1 :: 97] = 0  # rows of padding
  return x


def _pitch(k):
  return -(-k // 16) * 16


def _padded(values, k):
  """8-bit rows at a pitch of whole 16 bytes."""
  t = torch.zeros(values.shape[0], _pitch(k), dtype=torch.uint8, device="cuda")
  t[:, :k] = values.view(torch.uint8)
  return t.view(torch.float8_e4m3fn)


def prepare(case, seed):
  g = _generator(seed)
  if case["op"] == "quantize":
    rows, k, block = case["rows"], case["k"], case["block"]
    if block == 1:
      x = _activations(rows, k, g)
    else:
      x = torch.randn(rows, k, device="cuda", generator=g) * k**-0.5
    return dict(case, x=x.to(TYPES[case["type"]]), q=torch.empty(rows, _pitch(k), dtype=torch.float8_e4m3fn, device="cuda"),
                scale=torch.empty(-(-rows // block), -(-k // BLOCK), device="cuda"))
  if case["op"] == "linear":
    rows, k, n = case["rows"], case["k"], case["n"]
    s = dict(case, **{"out": torch.empty(rows, n, dtype=TYPES[case["out"]], device="cuda"), "out type": case["out"]})
    x = _activations(rows, k, g).to(torch.bfloat16 if case["x"] == "bf16" else torch.float32)
    s["x scale"] = None
    if case["x"] == "fp8":
      q, s["x scale"] = _quantised(x, 1)
      x = _padded(q, k)
    s["x"], s["x type"] = x, case["x"]
    q, s["w scale"] = _quantised(torch.randn(n, k, device="cuda", generator=g) * k**-0.5, BLOCK)
    s["w"] = _padded(q, k)
    s["scratch"] = torch.empty(rows * (_pitch(k) + 4 * -(-k // BLOCK)) + 4096, dtype=torch.uint8, device="cuda")
    return s
  if case["op"] == "control":
    return _control_state(case, g)
  slots, vocab, tokens = case["slots"], case["vocab"], case["tokens"]
  s = dict(case, seen=torch.zeros(slots, -(-vocab // 8) * 8, dtype=torch.int16, device="cuda"), touched=torch.zeros(slots, -(-vocab // 256), dtype=torch.int32, device="cuda"))
  s["token"] = _tokens(tokens, vocab, g)
  if tokens == slots:
    s["slot"] = torch.randperm(slots, device="cuda", generator=g).int()
  else:  # ragged prompts one behind the other
    s["slot"] = torch.randint(0, slots, (tokens,), device="cuda", generator=g).sort().values.int()
  s["slot"][tokens // 3 :: 50] = -1  # rows of the step that belong to nobody
  return s


def _tokens(count, vocab, g):
  """Token ids as texts have them: a few of them often, most of them seldom."""
  u = torch.rand(count, device="cuda", generator=g, dtype=torch.float64)
  return ((vocab**u - 1) / (vocab - 1) * vocab * 0.999).long().mul_(2654435761).remainder_(vocab).int()


def _control_state(case, g):
  rows, vocab, history, masks = case["rows"], case["vocab"], case["history"], case["masks"]
  slots = rows + 2
  s = dict(case, logits=4 * torch.randn(rows, vocab, device="cuda", generator=g), out=torch.empty(rows, vocab, device="cuda"))
  s["slot"] = torch.randperm(slots, device="cuda", generator=g)[:rows].int()
  seen = torch.zeros(slots * (-(-vocab // 8) * 8), dtype=torch.int32, device="cuda")
  at = torch.arange(slots, device="cuda").repeat_interleave(history) * (-(-vocab // 8) * 8) + _tokens(slots * history, vocab, g).long()
  new = torch.rand(slots * history, device="cuda", generator=g) < 0.6
  seen.index_add_(0, at[new], torch.ones_like(at[new], dtype=torch.int32))
  seen[at[~new]] |= 0x8000
  s["seen"] = torch.where(seen >= 0x8000, seen - 0x10000, seen).to(torch.int16).view(slots, -1)
  s["touched"] = _touched(s["seen"])
  s["repetition"] = 1 + torch.rand(slots, device="cuda", generator=g) * 9 * (torch.arange(slots, device="cuda") % 4 != 1)
  s["presence"] = torch.rand(slots, device="cuda", generator=g) * (torch.arange(slots, device="cuda") % 3 != 1)
  s["frequency"] = torch.rand(slots, device="cuda", generator=g) * 0.5 * (torch.arange(slots, device="cuda") % 3 != 2)
  s["bias off"] = s["bias token"] = s["bias value"] = None
  if case["biases"]:  # ascending and distinct in each row
    count = min(case["biases"], vocab // 2)
    first = torch.randint(0, vocab // count, (rows, count), device="cuda", generator=g)
    s["bias token"] = (first + torch.arange(count, device="cuda") * (vocab // count)).int().reshape(-1)
    s["bias value"] = 5 * torch.randn(rows * count, device="cuda", generator=g)
    s["bias off"] = torch.arange(0, rows * count + 1, count, device="cuda", dtype=torch.int32)
  s["allowed"] = s["allowed row"] = None
  if masks:
    # what may follow: a run of the vocabulary (audio tokens), scattered tokens (a grammar), and the last of several masks nothing
    t = torch.arange(-(-vocab // 32) * 32, device="cuda").view(1, -1, 32)
    kind = torch.arange(masks, device="cuda").view(-1, 1, 1)
    bits = torch.where(kind % 3 == 0, t >= vocab - vocab // 32, torch.rand(masks, t.shape[1], 32, device="cuda", generator=g) < 0.03)
    bits &= (kind < masks - 1) | (masks == 1)
    s["allowed"] = (bits.long() << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    s["allowed row"] = torch.where(torch.arange(rows, device="cuda") % 5 == 4, -1, torch.arange(rows, device="cuda") % max(1, masks - 1)).int()
    if masks > 1 and rows > 1:
      s["allowed row"][rows // 2] = masks - 1
  return s


# ---- the operators ---------------------------------------------------------------------------------------------------------------


def _quantised(x, block):
  """(values, scales) of x[rows, k]: blocks of `block` rows x 128 columns share amax / 448, and a value is x * (448 / amax), both fractions in 32 bits."""
  rows, k = x.shape
  up, blocks = -(-rows // block), -(-k // BLOCK)
  full = x.new_zeros(up * block, blocks * BLOCK, dtype=torch.float32)
  full[:rows, :k] = x
  full = full.view(up, block, blocks, BLOCK)
  largest = full.abs().amax((1, 3)).clamp(min=2.0**-96).double()  # (the fractions in 64 bits: a last bit of theirs moves values over a border)
  q = (full * (448 / largest).float()[:, None, :, None]).to(torch.float8_e4m3fn)
  return q.view(up * block, blocks * BLOCK)[:rows, :k], (largest / 448).float()


def _touched(seen):
  """Bit t / 8 of a slot's words is set where any of the eight tokens from t on has been seen."""
  slots, ld = seen.shape
  words = -(-ld // 256)
  any8 = torch.zeros(slots, words * 32, dtype=torch.bool, device=seen.device)
  any8[:, : ld // 8] = (seen.view(slots, -1, 8) != 0).any(-1)
  return (any8.view(slots, words, 32).long() << torch.arange(32, device=seen.device)).sum(-1).to(torch.int32)


def _spread(scale, block, rows, k):
  """One scale per value."""
  return scale.repeat_interleave(block, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :k]


def run(state):
  s = state
  if own:
    return _own(s)
  if s["op"] == "quantize":
    q, scale = _quantised(s["x"], s["block"])
    return dict(q=q, scale=scale)
  if s["op"] == "linear":
    rows, k, n = s["rows"], s["k"], s["n"]
    q, scale = (s["x"][:, :k], s["x scale"]) if s["x type"] == "fp8" else _quantised(s["x"], 1)
    x = q.float() * _spread(scale, 1, rows, k)
    return (x @ (s["w"][:, :k].float() * _spread(s["w scale"], BLOCK, n, k)).T).to(s["out"].dtype)
  if s["op"] == "control":
    slot = s["slot"].long()
    seen = s["seen"][slot, : s["vocab"]].int()
    count = (seen & 0x7FFF).float()
    l, repetition = s["logits"], s["repetition"][slot, None]
    l = torch.where(seen != 0, torch.where(l > 0, l / repetition, l * repetition), l)
    l = l - s["frequency"][slot, None] * count - s["presence"][slot, None] * (count > 0)
    if s["bias off"] is not None:
      row = torch.arange(s["rows"], device=l.device).repeat_interleave(len(s["bias token"]) // s["rows"])
      l.index_put_((row, s["bias token"].long()), s["bias value"], accumulate=True)
    if s["allowed"] is not None:
      bits = (s["allowed"][:, :, None] >> torch.arange(32, device=l.device, dtype=torch.int32)) & 1
      bits = bits.view(len(bits), -1)[:, : s["vocab"]].bool()
      at = s["allowed row"].long()
      l = torch.where(bits[at.clamp(min=0)] | (at < 0)[:, None], l, -math.inf)
    return l
  there = s["slot"] >= 0
  at = s["slot"].long().clamp(min=0) * s["seen"].shape[1] + s["token"]
  if s["prompt"]:
    noted = torch.zeros(s["seen"].numel(), dtype=torch.int32, device="cuda").index_put_((at,), there.int(), accumulate=True) > 0
    s["seen"] |= (noted.view(s["seen"].shape).int() << 15).to(torch.int16)
  else:
    more = torch.zeros(s["seen"].numel(), dtype=torch.int32, device="cuda").index_add_(0, at, there.int()).view(s["seen"].shape)
    count = ((s["seen"].int() & 0x7FFF) + more).clamp(max=0x7FFF)
    s["seen"].copy_((s["seen"].int() & ~0x7FFF) | count)
  s["touched"] |= _touched(s["seen"])
  return dict(seen=s["seen"], touched=s["touched"])


def _ptr(t):
  return 0 if t is None else t.data_ptr()


def _own(s):
  from maxtext_indextts2_b200 import _lib

  lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
  if s["op"] == "quantize":
    x, q = s["x"], s["q"]
    _lib.check(lib.mtx_quantize_fp8(x.data_ptr(), CODES[s["type"]], x.stride(0), s["rows"], s["k"], s["block"], q.data_ptr(), q.stride(0), s["scale"].data_ptr(), stream))
    return dict(q=q[:, : s["k"]], scale=s["scale"])
  if s["op"] == "linear":
    x, w, out, scratch = s["x"], s["w"], s["out"], s["scratch"]
    _lib.check(lib.mtx_linear_fp8(x.data_ptr(), CODES[s["x type"]], x.stride(0), _ptr(s["x scale"]), w.data_ptr(), w.stride(0), s["w scale"].data_ptr(), out.data_ptr(),
                                  CODES[s["out type"]], out.stride(0), s["rows"], s["n"], s["k"], scratch.data_ptr(), scratch.numel(), stream))
    return out
  if s["op"] == "control":
    seen, touched, allowed = s["seen"], s["touched"], s["allowed"]
    controls = _lib.LogitControls(
        slots=seen.shape[0], slot=s["slot"].data_ptr(), seen=seen.data_ptr(), ld_seen=seen.stride(0), touched=touched.data_ptr(), ld_touched=touched.stride(0),
        repetition=s["repetition"].data_ptr(), presence=s["presence"].data_ptr(), frequency=s["frequency"].data_ptr(),
        bias_off=_ptr(s["bias off"]), bias_token=_ptr(s["bias token"]), bias_value=_ptr(s["bias value"]),
        allowed_rows=0 if allowed is None else allowed.shape[0], allowed_row=_ptr(s["allowed row"]), allowed=_ptr(allowed), ld_allowed=0 if allowed is None else allowed.stride(0))
    logits, out = s["logits"], s["out"]
    _lib.check(lib.mtx_control_logits(logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0), s["rows"], s["vocab"], controls, stream))
    return out
  seen, touched, token = s["seen"], s["touched"], s["token"]
  _lib.check(lib.mtx_note_tokens(seen.data_ptr(), seen.stride(0), touched.data_ptr(), touched.stride(0), seen.shape[0], s["vocab"], token.data_ptr(), s["slot"].data_ptr(),
                                 len(token), int(s["prompt"]), stream))
  return dict(seen=seen, touched=touched)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------


def _e4m3(v):
  """The nearest value with four significant bits, exponents from -6 to 8, at most 448 in size; ties to the even one."""
  size = v.abs()
  _, e = torch.frexp(size)
  step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
  return torch.sign(v) * torch.minimum(torch.round(size / step) * step, torch.full_like(size, 448))


def _blockwise(x, block):
  """Values and scales of x in 64 bits, a column of blocks at a time; what the definition holds in 32 bits (the two fractions, the scaled value) is rounded to them."""
  rows, k = x.shape
  q, scales = torch.empty(rows, k, dtype=torch.float64, device=x.device), []
  group = torch.arange(rows, device=x.device) // block
  for c in range(0, k, BLOCK):
    part = x[:, c : c + BLOCK].double()
    largest = torch.full((-(-rows // block),), 2.0**-96, dtype=torch.float64, device=x.device).scatter_reduce_(0, group, part.abs().max(1).values, "amax")
    scales.append((largest / 448).float().double())
    q[:, c : c + BLOCK] = _e4m3((part * (448 / largest).float().double()[group, None]).float().double())
  return q, torch.stack(scales, 1)


def exact(case, seed):
  if case["op"] == "note":
    return None
  s = prepare(case, seed)
  if case["op"] == "quantize":
    q, scale = _blockwise(s["x"], s["block"])
    return dict(q=q, scale=scale)
  if case["op"] == "linear":
    k, n = s["k"], s["n"]
    q, scale = (s["x"][:, :k].double(), s["x scale"].double()) if s["x type"] == "fp8" else _blockwise(s["x"], 1)
    sums = torch.zeros(s["rows"], n, dtype=torch.float64, device="cuda")
    group = torch.arange(n, device="cuda") // BLOCK
    for b, c in enumerate(range(0, k, BLOCK)):
      sums += (q[:, c : c + BLOCK] @ s["w"][:, c : min(c + BLOCK, k)].double().T) * scale[:, b, None] * s["w scale"].double()[group, b]
    return sums
  out = s["logits"].double()
  lowest = torch.full((s["vocab"],), -math.inf, dtype=torch.float64, device="cuda")
  for r in range(s["rows"]):
    slot = int(s["slot"][r])
    word = s["seen"][slot, : s["vocab"]].long() & 0xFFFF
    hit = word.nonzero()[:, 0]
    times, old = (word[hit] & 0x7FFF).double(), out[r, hit]
    rep = s["repetition"][slot].double()
    out[r, hit] = old * torch.where(old > 0, 1 / rep, rep) - times * s["frequency"][slot].double() - times.clamp(max=1) * s["presence"][slot].double()
    if s["bias off"] is not None:
      b0, b1 = int(s["bias off"][r]), int(s["bias off"][r + 1])
      out[r].scatter_add_(0, s["bias token"][b0:b1].long(), s["bias value"][b0:b1].double())
    if s["allowed"] is not None and int(s["allowed row"][r]) >= 0:
      words = s["allowed"][int(s["allowed row"][r])].view(torch.uint8)  # eight tokens a byte, the lowest bit first
      may = torch.stack([words >> b & 1 for b in range(8)], 1).reshape(-1)[: s["vocab"]] != 0
      out[r] = torch.where(may, out[r], lowest)
  return out
