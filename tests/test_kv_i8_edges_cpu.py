"""Keys and values in 8 bits where a call is at its edges: what the library refuses, and what the CPU forms say. No GPU is needed."""

import pytest
import torch

from parallax_b200 import ops
from parallax_b200.ops import KernelError, _lib, cuda as cu
from tests.helpers import kv_i8_oracle as oracle

INVALID_ARG = 1
P = 1 << 20        # an address that nothing reads: every call below is refused


def _library():
    if not _lib.available():
        pytest.skip("the kernel library is not built")
    return _lib.lib()


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
def test_magnitudes_that_start_on_no_8_bytes_are_refused(D, page):
    """They are read in pairs: by the read-out and the eviction as by the attentions."""
    lib = _library()
    tail = (2, D, page, 4, 64, None, None)
    assert lib.pxl_kv_i8_load(P, P, P + 4, P, P, P, P, 3, 1, *tail) == INVALID_ARG
    assert lib.pxl_kv_i8_evict(P, P, P + 4, P, 64, 1, None, P, P, P, P, P, 1, 2, D, page, 4, 2, 64, 30, 2, 2, None, None) == INVALID_ARG
