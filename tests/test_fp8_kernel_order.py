"""The products' kernels start before the kernel in front is done.  What none of their warps may do before then, read from their source (a kernel in front
that takes seconds has no place in a test)."""

import os
import re

import pytest

from maxtext_indextts2_b200 import _lib

KERNELS = ["fp8_stream_kernel", "fp8_pair_kernel", "fp8_tile_kernel"]


def roles(name):
  """The kernel's text in front of the warps' roles, and each role's."""
  with open(os.path.join(_lib.CSRC, "fp8_linear.cuh"), encoding="utf-8") as f:
    text = f.read()
  start = re.search(name + r"\(const __grid_constant__", text).start()
  body = text[start : text.index("\n}\n", start)]
  first = re.search(r"^  if \(warp (==|>=) \d\) \{\n(?:(?!^  \}).*\n)*?^  \} else", body, re.M).start()  # (the first choice by warp that has another side)
  last = body.index("\n  }\n", first)
  return body[:first], re.split(r"^  \} else (?:if \([^\n]*\) )?\{\n", body[first:last], flags=re.M)


@pytest.mark.parametrize("name", KERNELS)
def test_limited_waits_begin_behind_the_kernel_in_front(name):
  """A wait that gives up after some time counts its own kernel's time alone."""
  front, parts = roles(name)
  assert len(parts) == 3 and sum("fp8_wait(" in p for p in parts) == 3
  assert "fp8_wait(" not in front
  for part in parts:
    assert "griddep_wait();" in front or part.index("griddep_wait();") < part.index("fp8_wait("), part[:200]


@pytest.mark.parametrize("file", ["fp8_linear.cuh", "logit_controls.cuh"])
def test_nothing_is_read_by_the_read_only_path(file):
  """That path is for what nobody writes while the kernel lives; the kernel in front may still write all that these read."""
  with open(os.path.join(_lib.CSRC, file), encoding="utf-8") as f:
    code = re.sub(r"//.*", "", f.read())
  assert re.findall(r"__ldg\b|global\.nc|__restrict__", code) == []
