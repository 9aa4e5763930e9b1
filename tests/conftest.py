"""pytest configuration: the ``gpu`` marker and import paths."""

import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
  sys.path.insert(0, ROOT)


def pytest_configure(config):
  config.addinivalue_line("markers", "gpu: needs a CUDA device (run on the B200 box with -m gpu)")


def pytest_collection_modifyitems(config, items):
  try:
    import torch

    has_gpu = torch.cuda.is_available()
  except Exception:  # pragma: no cover
    has_gpu = False
  if has_gpu:
    return
  skip = pytest.mark.skip(reason="no CUDA device in this container")
  for item in items:
    if "gpu" in item.keywords:
      item.add_marker(skip)


@pytest.fixture(autouse=True)
def _no_stalled_products(request):
  """Behind every test of 8-bit products: no wait in their kernels has run out (their results would be wrong without an error)."""
  yield
  if "gpu" in request.keywords and request.module.__name__.rpartition(".")[2] in ("test_fp8_linear_gpu", "test_answer_step_gpu", "test_far_offsets_gpu"):
    import ctypes

    from maxtext_indextts2_b200 import _lib

    count = ctypes.c_uint32(1)
    _lib.check(_lib.load().mtx_linear_fp8_stalls(ctypes.byref(count)))
    assert count.value == 0
