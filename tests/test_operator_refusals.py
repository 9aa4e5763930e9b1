"""What the 8-bit products and the logit controls refuse; none of it reaches a GPU."""

import pytest

from maxtext_indextts2_b200 import _lib

A = 1 << 20  # an address that is aligned like device memory; every call below is refused before it is looked at


@pytest.fixture(scope="module")
def lib():
  _lib.build()
  return _lib.load()


def refused(rc, word):
  assert rc == _lib.MTX_ERR_ARG and word in _lib.last_error(), (rc, _lib.last_error())


QUANT = dict(x=A, x_type=_lib.BF16, ldx=256, rows=4, k=256, block_rows=1, q=A, ldq=256, scale=A, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x_type=_lib.E4M3), "x_type"), (dict(x_type=9), "x_type"), (dict(block_rows=64), "block_rows"), (dict(rows=-1), "bad rows"), (dict(k=0), "bad rows"),
    (dict(ldx=255), "bad rows"), (dict(ldq=255), "bad rows"), (dict(k=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31), "bad rows"), (dict(x=None), "null"), (dict(q=None), "null"),
    (dict(scale=None), "null"), (dict(q=A + 8), "16-byte"), (dict(x=A + 1), "multiples"), (dict(x=A + 2, x_type=_lib.F32), "multiples"), (dict(scale=A + 2), "multiples"),
    (dict(ldq=264), "16"), (dict(rows=1 << 30, k=1024, ldx=1024, ldq=1024), "2^31"), (dict(rows=(1 << 30) + 1, k=16, ldx=16, ldq=16), "bad rows"),
])
def test_quantize(lib, change, word):
  refused(lib.mtx_quantize_fp8(*{**QUANT, **change}.values()), word)


LINEAR = dict(x=A, x_type=_lib.BF16, ldx=256, x_scale=None, wq=A, ldw=256, w_scale=A, out=A, out_type=_lib.BF16, ldo=128, rows=4, n=128, k=256, scratch=A, scratch_bytes=1 << 20,
              stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(x_type=3), "x_type"), (dict(out_type=_lib.E4M3), "out_type"), (dict(rows=-1), "bad rows"), (dict(n=0), "bad rows"), (dict(k=0), "bad rows"), (dict(ldx=255), "bad rows"),
    (dict(ldw=255), "bad rows"), (dict(ldo=127), "bad rows"), (dict(x=None), "null"), (dict(wq=None), "null"), (dict(w_scale=None), "null"), (dict(out=None), "null"),
    (dict(x_type=_lib.E4M3), "null"), (dict(wq=A + 4), "16-byte"), (dict(ldw=260), "16-byte"), (dict(x_type=_lib.E4M3, x_scale=A, x=A + 1), "16-byte"),
    (dict(x=A + 1), "multiples"), (dict(out=A + 1), "multiples"), (dict(out=A + 2, out_type=_lib.F32), "multiples"), (dict(w_scale=A + 2), "multiples"),
    (dict(x_type=_lib.E4M3, x_scale=A + 1), "multiples"), (dict(scratch=None), "scratch"), (dict(scratch=A + 4), "scratch"), (dict(scratch_bytes=100), "scratch"), (dict(rows=1 << 30, k=1024, ldx=1024, ldw=1024), "2^31"), (dict(rows=(1 << 30) + 1), "bad rows"), (dict(n=(1 << 30) + 1, ldo=1 << 31), "bad rows"),
])
def test_linear(lib, change, word):
  refused(lib.mtx_linear_fp8(*{**LINEAR, **change}.values()), word)


def test_scratch_of_a_linear(lib):
  assert lib.mtx_linear_fp8_scratch_bytes(0, 5) == 0 and lib.mtx_linear_fp8_scratch_bytes(5, 0) == 0
  need = lib.mtx_linear_fp8_scratch_bytes(3, 130)
  assert need >= 3 * 144 + 3 * 2 * 4


def test_stalls(lib):
  refused(lib.mtx_linear_fp8_stalls(None), "null")


CONTROL = dict(logits=A, ld=64, out=A + 65536, ldo=64, rows=2, vocab=64, controls=None, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "bad rows"), (dict(vocab=0), "bad rows"), (dict(ld=63), "bad rows"), (dict(ldo=63), "bad rows"), (dict(vocab=(1 << 28) + 1, ld=1 << 31, ldo=1 << 31), "bad rows"),
    (dict(logits=None), "null"), (dict(out=None), "null"), (dict(out=A, ldo=72), "in place"), (dict(out=A + 2), "4 bytes"), (dict(logits=A + 1), "4 bytes"),
])
def test_control(lib, change, word):
  refused(lib.mtx_control_logits(*{**CONTROL, "controls": _lib.LogitControls(), **change}.values()), word)


def test_control_without_controls(lib):
  refused(lib.mtx_control_logits(A, 64, A, 64, 2, 64, None, None), "null controls")


def test_no_rows_is_no_error(lib):
  assert lib.mtx_control_logits(None, 64, None, 64, 0, 64, _lib.LogitControls(), None) == _lib.MTX_OK
  assert lib.mtx_quantize_fp8(None, 0, 64, 0, 64, 1, None, 64, None, None) == _lib.MTX_OK
  assert lib.mtx_linear_fp8(None, 0, 64, None, None, 64, None, None, 0, 64, 0, 64, 64, None, 0, None) == _lib.MTX_OK
  assert lib.mtx_note_tokens(None, 64, None, 0, 1, 64, None, None, 0, 0, None) == _lib.MTX_OK


@pytest.mark.parametrize("fields,word", [
    (dict(repetition=A), "need the record"), (dict(seen=A, slots=0, ld_seen=64), "record"), (dict(seen=A, slots=1, ld_seen=60), "record"), (dict(seen=A, slots=1, ld_seen=68), "record"),
    (dict(seen=A + 2, slots=1, ld_seen=64), "record"), (dict(seen=A, slots=1, ld_seen=64, touched=A), "touched"), (dict(bias_off=A), "together"), (dict(bias_token=A, bias_value=A), "together"),
    (dict(slot=A + 1), "4 bytes"), (dict(seen=A, slots=1, ld_seen=64, presence=A + 2), "4 bytes"), (dict(bias_off=A, bias_token=A + 2, bias_value=A), "4 bytes"),
    (dict(allowed=A + 1, allowed_rows=1, ld_allowed=2), "4 bytes"), (dict(allowed=A, ld_allowed=2), "allowed"), (dict(allowed=A, allowed_rows=1, ld_allowed=1), "allowed"),
])
def test_fields_of_the_controls(lib, fields, word):
  refused(lib.mtx_control_logits(*{**CONTROL, "controls": _lib.LogitControls(**fields)}.values()), word)


NOTE = dict(seen=A, ld_seen=64, touched=A, ld_touched=1, slots=4, vocab=64, token=A, slot=A, n=4, prompt=0, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(n=-1), "bad n"), (dict(vocab=0), "bad n"), (dict(vocab=(1 << 28) + 8, ld_seen=1 << 31, ld_touched=1 << 24), "bad n"), (dict(seen=None), "null"), (dict(token=None), "null"),
    (dict(slot=None, n=5), "slot i"), (dict(ld_seen=56), "record"), (dict(seen=A + 8), "record"), (dict(slots=0), "record"), (dict(ld_touched=0), "touched"), (dict(touched=A + 2), "touched"), (dict(token=A + 2), "4 bytes"), (dict(slot=A + 1), "4 bytes"),
])
def test_note(lib, change, word):
  refused(lib.mtx_note_tokens(*{**NOTE, **change}.values()), word)
