"""What the operators of a step of drafted tokens refuse, and the frequencies of rotary positions; none of it reaches a GPU."""

import ctypes
import math
import pathlib

import pytest

from maxtext_indextts2_b200 import _lib, fibelix

A = 1 << 20  # an address that is aligned like device memory; every call below is refused before it is looked at


@pytest.fixture(scope="module")
def lib():
  _lib.build()
  return _lib.load()


def refused(rc, word, code=_lib.MTX_ERR_ARG):
  assert rc == code and word in _lib.last_error(), (rc, _lib.last_error())


NORM = dict(x=A, x_type=_lib.BF16, ldx=256, residual=A, residual_type=_lib.BF16, ld_residual=256, sum=A + 65536, ld_sum=256, weight=A, weight_type=_lib.F32, weight_offset=0.0, eps=1e-5,
            out=A + 131072, out_type=_lib.E4M3, ldo=256, out_scale=A, rows=4, width=256, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x_type=_lib.E4M3), "x_type"), (dict(residual_type=2), "residual_type"), (dict(weight_type=7), "weight_type"), (dict(out_type=3), "out_type"), (dict(rows=-1), "bad rows"),
    (dict(rows=(1 << 30) + 1), "bad rows"), (dict(width=0), "bad rows"), (dict(width=32769, ldx=1 << 16, ld_residual=1 << 16, ld_sum=1 << 16, ldo=1 << 16), "bad rows"), (dict(ldx=255), "bad rows"), (dict(ld_residual=255), "bad rows"),
    (dict(ld_sum=255), "bad rows"), (dict(ldo=255), "bad rows"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(residual=None), "needs a residual"), (dict(x=None), "null"),
    (dict(out=None), "null"), (dict(out_scale=None), "null"), (dict(out=A + 8), "16-byte"), (dict(ldo=264), "16-byte"), (dict(x=A + 1), "multiples"),
    (dict(residual=A + 2, residual_type=_lib.F32), "multiples"), (dict(sum=A + 1), "multiples"), (dict(weight=A + 2), "multiples"), (dict(out=A + 2, out_type=_lib.F32), "multiples"),
    (dict(out_scale=A + 2), "multiples"), (dict(sum=A + 65536, out=A + 65536, out_type=_lib.BF16), "two results"), (dict(sum=A, ld_sum=512), "type and pitch"),
    (dict(out=A, out_type=_lib.F32, sum=None, residual=None), "type and pitch"), (dict(out=A), "type and pitch"), (dict(x=A + 65536, ldx=264), "type and pitch"),
])
def test_norm(lib, change, word):
  refused(lib.mtx_add_rmsnorm(*{**NORM, **change}.values()), word)


def test_nothing_is_no_error(lib):
  assert lib.mtx_add_rmsnorm(*{**NORM, "rows": 0, "x": None}.values()) == _lib.MTX_OK
  assert lib.mtx_rotary(_lib.RotaryBatch(**{**ROTARY, "rows": 0, "q": None}), None) == _lib.MTX_OK
  for change in (dict(rows=0), dict(sequences=0, prefixes=0)):
    assert attend(lib, **change) == _lib.MTX_OK
  assert verify(lib, sequences=0) == _lib.MTX_OK


ROTARY = dict(rows=4, heads=4, kv_heads=2, dim=64, rot_dims=64, rot_half=0, amplitude=1.0, type=_lib.BF16, out_type=_lib.BF16, freq=A, pos=A, q=A, k=A, v=A, ldq=256, ldk=128, ldv=128,
              q_out=A + 65536, ldq_out=256, k_out=A + 131072, ldk_out=128)
PAGES = dict(k_pages=A, v_pages=A, groups=4, num_pages=8, tokens_per_page=16, max_pages_per_group=2, group=A, page_map=A)


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "bad rows"), (dict(rows=(1 << 30) + 1), "bad rows"), (dict(heads=-1), "bad rows"), (dict(heads=0, kv_heads=0), "bad rows"), (dict(dim=0), "bad rows"), (dict(dim=1025), "bad rows"), (dict(rot_dims=66), "bad rows"),
    (dict(rot_dims=3), "bad rows"), (dict(rot_dims=-2), "bad rows"), (dict(type=2), "type"), (dict(out_type=2), "type"), (dict(ldq=255), "pitches"), (dict(ldk=127), "pitches"),
    (dict(ldq_out=255), "pitches"), (dict(ldk_out=127), "pitches"), (dict(pos=None), "null"), (dict(freq=None), "null"), (dict(q=None), "null"), (dict(q_out=None), "null"), (dict(k=None), "null"),
    (dict(k_out=None), "null"), (dict(q=A + 1), "multiples"), (dict(k_out=A + 1), "multiples"), (dict(pos=A + 2), "multiples"), (dict(freq=A + 4), "multiples"),
    (dict(q_out=A, ldq_out=320), "type and pitch"), (dict(k_out=A, out_type=_lib.F32), "type and pitch"), (dict(k_pages=A), "together"), (dict(**{**PAGES, "page_map": None}), "together"),
    (dict(**{**PAGES, "groups": 0}), "groups / pages"), (dict(**{**PAGES, "num_pages": 0}), "groups / pages"), (dict(**{**PAGES, "tokens_per_page": 0}), "groups / pages"),
    (dict(**{**PAGES, "max_pages_per_group": 0}), "groups / pages"), (dict(**{**PAGES, "group": None, "groups": 3}), "row r belongs"), (dict(**PAGES, ldv=127), "pitches"),
    (dict(**PAGES, v=None), "null"), (dict(**{**PAGES, "k_pages": A + 1}), "multiples"), (dict(**{**PAGES, "page_map": A + 1}), "multiples"),
    (dict(**{**PAGES}, kv_heads=0), "groups / pages"),
])
def test_rotary(lib, change, word):
  refused(lib.mtx_rotary(_lib.RotaryBatch(**{**ROTARY, **change}), None), word)


def test_rotary_without_a_batch(lib):
  refused(lib.mtx_rotary(None, None), "null batch")


def frequencies(lib, dims, base, kind, factor=0.0, original=0.0, low=0.0, high=0.0):
  freq, amplitude = (ctypes.c_double * max(1, dims // 2))(), ctypes.c_float(-1)
  _lib.check(lib.mtx_rotary_frequencies(dims, base, _lib.ROTARY[kind], factor, original, low, high, freq, ctypes.byref(amplitude)))
  return list(freq), amplitude.value


@pytest.mark.parametrize("dims,base", [(2, 1e4), (64, 1e4), (50, 5e5), (256, 1e6)])
def test_frequencies(lib, dims, base):
  plain = [base ** (-2 * i / dims) for i in range(dims // 2)]
  near = lambda a, b: all(abs(x - y) <= 1e-13 * abs(y) for x, y in zip(a, b))
  got, one = frequencies(lib, dims, base, "plain")
  assert near(got, plain) and one == 1.0
  got, one = frequencies(lib, dims, base, "linear", 8.0)
  assert near(got, [f / 8 for f in plain]) and one == 1.0
  got, one = frequencies(lib, dims, base, "bands", 8.0, 8192.0, 1.0, 4.0)
  for f, g in zip(plain, got):
    turns = 8192 * f / (2 * math.pi)
    part = min(1.0, max(0.0, (turns - 1.0) / 3.0))
    assert abs(g - (f * part + f / 8 * (1 - part))) <= 1e-13 * g
  assert one == 1.0
  got, one = frequencies(lib, dims, base, "yarn", 4.0, 2048.0, 1.0, 32.0)
  want, amplitude = fibelix.yarn_rot_frequencies(dims, base, dict(factor=4.0, original=2048.0, fast=32.0, slow=1.0))
  assert near(got, want.tolist()) and abs(one - amplitude) < 1e-6


@pytest.mark.parametrize("args,word", [
    ((0, 1e4, 0, 1.0, 1.0, 1.0, 2.0), "rot_dims"), ((7, 1e4, 0, 1.0, 1.0, 1.0, 2.0), "rot_dims"), ((64, 1.0, 0, 1.0, 1.0, 1.0, 2.0), "rot_dims"), ((64, math.inf, 0, 1.0, 1.0, 1.0, 2.0), "rot_dims"),
    ((64, 1e4, 4, 1.0, 1.0, 1.0, 2.0), "scaling"), ((64, 1e4, -1, 1.0, 1.0, 1.0, 2.0), "scaling"), ((64, 1e4, 1, 0.5, 1.0, 1.0, 2.0), "factor"), ((64, 1e4, 1, math.nan, 1.0, 1.0, 2.0), "factor"),
    ((64, 1e4, 2, 2.0, 0.0, 1.0, 2.0), "borders"), ((64, 1e4, 3, 2.0, 100.0, 2.0, 2.0), "borders"), ((64, 1e4, 3, 2.0, 100.0, 0.0, 2.0), "borders"),
])
def test_frequencies_refused(lib, args, word):
  freq, amplitude = (ctypes.c_double * 32)(), ctypes.c_float()
  refused(lib.mtx_rotary_frequencies(*args, freq, ctypes.byref(amplitude)), word)
  refused(lib.mtx_rotary_frequencies(64, 1e4, 0, 1.0, 1.0, 1.0, 2.0, None, ctypes.byref(amplitude)), "null")


BATCH = dict(rows=4, sequences=2, row0=A, lengths=A, page_map=A, prefixes=1, prefix_seq0=A, prefix_len=A)
ATTEND = dict(q=A, ldq=256, k_pages=A, v_pages=A, batch=None, out=A, ldo=256, num_q_heads=4, num_kv_heads=2, head_dim=64, num_pages=8, tokens_per_page=16, max_pages_per_group=4, scale=0.125,
              softcap=0.0, scratch=A, scratch_bytes=1 << 30, stream=None)


def attend(lib, **change):
  batch = _lib.PrefixBatch(**{k: change.pop(k, v) for k, v in BATCH.items()})
  return lib.mtx_prefix_attention(*{**ATTEND, "batch": batch, **change}.values())


@pytest.mark.parametrize("change,word", [
    (dict(num_pages=0), "page counts"), (dict(max_pages_per_group=0), "page counts"), (dict(max_pages_per_group=1 << 26, tokens_per_page=16), "page counts"), (dict(rows=-1), "bad rows"),
    (dict(rows=(1 << 20) + 1), "bad rows"), (dict(sequences=-1), "bad rows"), (dict(sequences=(1 << 16) + 1), "bad rows"), (dict(prefixes=-1), "bad rows"), (dict(prefixes=3), "bad rows"),
    (dict(ldq=255), "pitches"), (dict(ldo=248), "pitches"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(softcap=-1.0), "scale"),
    (dict(softcap=math.inf), "scale"), (dict(q=None), "null"), (dict(k_pages=None), "null"), (dict(v_pages=None), "null"), (dict(out=None), "null"), (dict(row0=None), "null"),
    (dict(lengths=None), "null"), (dict(page_map=None), "null"), (dict(prefix_seq0=None), "null"), (dict(prefix_len=None), "null"), (dict(q=A + 2), "16 bytes"), (dict(ldq=260), "16 bytes"),
    (dict(out=A + 8), "16 bytes"), (dict(ldo=268), "16 bytes"), (dict(k_pages=A + 8), "16 bytes"), (dict(row0=A + 2), "4 bytes"), (dict(prefix_len=A + 1), "4 bytes"), (dict(scratch=None), "scratch"),
    (dict(scratch=A + 16), "scratch"), (dict(scratch_bytes=10), "scratch"),
])
def test_attention(lib, change, word):
  refused(attend(lib, **change), word)


@pytest.mark.parametrize("change,word", [
    (dict(head_dim=96), "head_dim"), (dict(num_q_heads=5), "query heads"), (dict(num_q_heads=34, ldq=1 << 14, ldo=1 << 14), "query heads"), (dict(num_kv_heads=0), "query heads"),
    (dict(tokens_per_page=4), "tokens_per_page"), (dict(tokens_per_page=24), "tokens_per_page"), (dict(num_pages=1 << 27), "too many rows"),
])
def test_attention_unsupported(lib, change, word):
  refused(attend(lib, **change), word, _lib.MTX_ERR_UNSUPPORTED)


def test_attention_without_a_batch(lib):
  refused(lib.mtx_prefix_attention(*ATTEND.values()), "null batch")


def test_stalls(lib):
  refused(lib.mtx_prefix_attention_stalls(None), "null")


def test_scratch_of_an_attention(lib):
  size = lib.mtx_prefix_attention_scratch_bytes
  assert size(0, 1, 0, 4, 2, 64) == 0 and size(4, 0, 0, 4, 2, 64) == 0 and size(4, 1, -1, 4, 2, 64) == 0
  assert 0 < size(4, 2, 1, 4, 2, 64) <= size(400, 20, 3, 16, 4, 128)


DRAFT = dict(rows=4, sequences=2, vocab=64, row0=A, token=A, target=A, ld_target=64, draft=A, ld_draft=64, temperature=A, draft_temperature=A, accept_u=A, pick_u=A)


def verify(lib, accepted=A, emitted=A, scratch=A, scratch_bytes=1 << 30, **change):
  return lib.mtx_verify_drafts(_lib.DraftBatch(**{**DRAFT, **change}), accepted, emitted, scratch, scratch_bytes, None)


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "bad rows"), (dict(rows=(1 << 20) + 1), "bad rows"), (dict(sequences=-1), "bad rows"), (dict(sequences=(1 << 16) + 1), "bad rows"), (dict(vocab=0), "bad rows"),
    (dict(vocab=(1 << 28) + 1, ld_target=1 << 30, ld_draft=1 << 30), "bad rows"), (dict(ld_target=63), "bad rows"), (dict(ld_draft=63), "bad rows"), (dict(accepted=None), "null"),
    (dict(emitted=None), "null"), (dict(row0=None), "null"), (dict(token=None), "null"), (dict(target=None), "null"), (dict(accept_u=None), "null"), (dict(pick_u=None), "null"),
    (dict(target=A + 2), "4 bytes"), (dict(draft=A + 1), "4 bytes"), (dict(emitted=A + 2), "4 bytes"), (dict(scratch=None), "scratch"), (dict(scratch=A + 8), "scratch"),
    (dict(scratch_bytes=8), "scratch"),
])
def test_verification(lib, change, word):
  refused(verify(lib, **change), word)


def test_verification_without_a_batch(lib):
  refused(lib.mtx_verify_drafts(None, A, A, A, 1 << 20, None), "null batch")


def test_scratch_of_a_verification(lib):
  size = lib.mtx_verify_drafts_scratch_bytes
  assert size(0, 1, 64) == 0 and size(4, 0, 64) == 0 and size(4, 2, 0) == 0 and 0 < size(4, 2, 64) <= size(40, 8, 264192)


def test_scratch_of_smaller_attentions(lib):
  """What the largest step has is enough for every smaller one, on either side of where prefixes get a kernel of their own."""
  size = lib.mtx_prefix_attention_scratch_bytes
  steps = [1, 2, 5, 16, 20, 39, 40, 41, 64, 65, 128, 319, 320, 321, 1000, 65536]
  for heads, kv, dim in ((16, 4, 128), (4, 4, 64), (16, 1, 256), (20, 4, 64)):
    for rows in steps:
      for sequences in steps[:9]:
        prefixes = [size(rows, sequences, n, heads, kv, dim) for n in range(sequences + 1)]
        assert prefixes == sorted(prefixes)
    for sequences in (1, 64, 65536):
      for prefixes in (0, 1, 40, 65536):
        rows = [size(n, sequences, min(prefixes, sequences), heads, kv, dim) for n in steps]
        assert rows == sorted(rows)
        assert size(320, sequences, min(prefixes, sequences), heads, kv, dim) <= size(320, sequences + 1, min(prefixes, sequences), heads, kv, dim)


def test_scratch_of_smaller_verifications(lib):
  """Chunks get larger from some rows on, and a call needs less: what the largest step has is enough all the same."""
  size = lib.mtx_verify_drafts_scratch_bytes
  for vocab in (1, 1000, 32768, 50000, 65536, 65537, 128000, 264192, 1 << 20, 1 << 28):
    rows = [size(n, 64, vocab) for n in list(range(1, 1300)) + [4000, 1 << 16, 1 << 20]]
    assert rows == sorted(rows)
    assert [size(100, n, vocab) for n in (1, 5, 64, 65535)] == sorted(size(100, n, vocab) for n in (1, 5, 64, 65535))
  for n in (1, 33, 34, 320, 1095, 1100, 1 << 20):
    tokens = [size(n, 64, v) for v in list(range(1, 300000, 997)) + [1 << 20, 1 << 24, 1 << 28]]
    assert tokens == sorted(tokens)


def test_tensor_memory_is_taken_behind_the_wait():
  """All columns taken before the kernels in front are through: one of those that starts its successor before it has its own columns would never get them, and neither kernel would end."""
  source = (pathlib.Path(_lib.__file__).parent / "csrc" / "prefix_attention.cuh").read_text()
  body = source[source.index("\nprefix_tc_kernel(") :]
  body = body[: body.index("\n}\n")]
  assert body.index("griddep_wait()") < body.index("tmem_alloc(") < body.index("griddep_launch_dependents()")
