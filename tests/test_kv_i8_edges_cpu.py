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


# ------------------------------------------------------------------------------------------------ more new tokens than a call says
@pytest.mark.parametrize("most", [0, 4])
def test_more_new_tokens_than_the_call_says_are_refused(most):
    """The forms that know the lengths when they are called refuse them before anything is written; the kernels report them."""
    g = torch.Generator().manual_seed(1)
    cache = oracle.make_cache(g, 4, 2, 16, 64)
    before = [c.clone() for c in cache]
    tab, ends, lens = torch.tensor([[0], [1]]).int(), torch.tensor([0, 2, 7]).int(), torch.tensor([9, 5]).int()
    x = torch.randn(7, 2, 64, generator=g).bfloat16()
    with pytest.raises(KernelError, match="max_q_len"):
        ops.store_kv_i8(x, x, *cache, tab, ends, lens, most)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    weights, out = torch.zeros(2, 2, 16), torch.full((7, 2, 64), 7.0).bfloat16()
    with pytest.raises(KernelError, match="max_q_len"):
        ops.attn_prefill_i8(x, *cache, tab, ends, lens, most, 0.1, out=out, weights=weights)
    assert (weights == 0).all() and (out == 7).all()
    with pytest.raises(KernelError, match="max_q_len"):
        ops.attn_prefill_i8(x, *cache, tab, ends, lens, -1, 0.1)


def test_calls_that_allow_no_new_tokens_reach_the_library(monkeypatch):
    """Sequences that have some all the same are reported there."""
    import contextlib

    calls = []

    class Recorder:
        def __getattr__(self, name):
            return lambda *args: calls.append(name) or 0

    monkeypatch.setattr(_lib, "lib", lambda: Recorder())
    monkeypatch.setattr(cu, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(cu, "_stream", lambda device: 0)
    monkeypatch.setattr(cu, "status_tensor", lambda device: torch.zeros(1, dtype=torch.int32))
    cache = oracle.make_cache(torch.Generator().manual_seed(2), 4, 2, 16, 64)
    x, tab, ends, lens = torch.zeros(3, 2, 64).bfloat16(), torch.zeros(1, 1).int(), torch.tensor([0, 3]).int(), torch.tensor([5]).int()
    cu.store_kv_i8(x, x, *cache, tab, ends, lens, 0)
    cu.attn_prefill_i8(x, *cache, tab, ends, lens, 0, 0.1)
    assert "pxl_kv_i8_store" in calls and "pxl_attn_i8_prefill" in calls
    with pytest.raises(KernelError, match="max_q_len"):
        cu.attn_prefill_i8(x, *cache, tab, ends, lens, -1, 0.1)


def test_a_negative_number_of_new_tokens_is_refused_by_the_library():
    lib = _library()
    sizes = (4, 2, 64, 16, 8, 8, 0.1, 0, 100, None, None)
    assert lib.pxl_kv_i8_store(P, P, 128, 128, P, P, P, P, P, P, 3, 1, -1, 2, 64, 16, 4, 4, None, None) == INVALID_ARG
    assert lib.pxl_attn_i8_prefill(P, 256, P, P, P, P, P, P, P, 256, None, None, P, 1 << 30, 2, 1, -1, *sizes) == INVALID_ARG
    assert lib.pxl_attn_i8_weigh(P, 256, P, P, P, P, P, P, P, 100, 1, None, P, 1 << 30, 2, 1, -1, *sizes) == INVALID_ARG
    assert lib.pxl_attn_i8_prefill_workspace(3, 1, 0, 4, 2, 64, 4096) >= lib.pxl_attn_i8_prefill_workspace(3, 1, 1, 4, 2, 64, 4096) > 0


# ------------------------------------------------------------------------------------------------ more new tokens than tokens
@pytest.mark.parametrize("n,t", [(5, 3), (5, 0), (40, 20), (33, 32)])
def test_store_of_more_new_tokens_than_tokens(n, t):
    """Those at positions below zero are left out; nothing but the sequence's pages is written."""
    g = torch.Generator().manual_seed(3)
    cache = oracle.make_cache(g, 5, 2, 16, 64)
    want = [c.clone() for c in cache]
    tab, k, v = torch.tensor([[0, 1, 2, 3]]).int(), torch.randn(n, 2, 64, generator=g).bfloat16(), torch.randn(n, 2, 64, generator=g).bfloat16()
    ops.store_kv_i8(k, v, *cache, tab, torch.tensor([0, n]).int(), torch.tensor([t]).int(), n)
    ops.store_kv_i8(k[n - t:], v[n - t:], *want, tab, torch.tensor([0, t]).int(), torch.tensor([t]).int(), n)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


# ------------------------------------------------------------------------------------------------ codes next to a tie
@pytest.mark.parametrize("x,m,want", [(129 / 32768, 1.0, 0), (1.0, 254.0, 0), (129 / 128, 254.0, 1), (3.0, 254.0, 2), (255 / 512, 127.0, 0),
                                      (64.0, 128.0, 64), (127.0, 254.0, 64), (129 / 256, 127.0, 1)])
def test_codes_of_numbers_next_to_a_tie(x, m, want):
    """127 x / m: 0.49998, 0.5, 0.504, 1.5, 0.498, 63.5, 63.5, 0.504."""
    cache = [torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1, 2)]
    k = torch.zeros(1, 1, 64)
    k[0, 0, :3] = torch.tensor([m, x, -x])
    assert torch.equal(k.bfloat16().float(), k)
    ops.store_kv_i8(k.bfloat16(), -k.bfloat16(), *cache, torch.zeros(1, 1).int(), torch.tensor([0, 1]).int(), torch.tensor([1]).int(), 1)
    assert cache[0][0, 0, 0, :3].tolist() == [127, want, -want] and cache[1][0, 0, 0, :3].tolist() == [-127, -want, want]


# ------------------------------------------------------------------------------------------------ results over queries
@pytest.mark.parametrize("shift", [0, 8, 128])
def test_results_over_the_queries_of_a_single_head_are_refused(shift):
    """Whatever the stride of a dimension of one says."""
    g = torch.Generator().manual_seed(4)
    cache = oracle.make_cache(g, 4, 1, 16, 64)
    flat = torch.randn(4 * 128, generator=g).bfloat16()
    tab, lens = torch.zeros(3, 1).int(), torch.ones(3).int()
    for stride in (64, 7, 3 * 128):
        q = flat.as_strided((3, 1, 64), (128, stride, 1))
        with pytest.raises(KernelError, match="overlaps the queries"):
            ops.attn_decode_i8(q, *cache, tab, lens, 0.1, out=flat.as_strided((3, 1, 64), (128, 64, 1), shift))
        ops.attn_decode_i8(q.clone(), *cache, tab, lens, 0.1, out=flat.as_strided((3, 1, 64), (128, 64, 1), 64))


# ------------------------------------------------------------------------------------------------ pages of zeros
def test_codes_of_a_page_whose_magnitude_stays_are_left_as_they_are():
    """Of a magnitude of zero too, where a caller's codes are any: they stand for zeros."""
    g = torch.Generator().manual_seed(5)
    cache = oracle.make_cache(g, 4, 2, 16, 64)
    cache[2][0] = 0.0
    before = [c.clone() for c in cache]
    x, ends = torch.zeros(1, 2, 64).bfloat16(), torch.tensor([0, 1]).int()
    ops.store_kv_i8(x, x, *cache, torch.zeros(1, 1).int(), ends, torch.tensor([6]).int(), 1)
    for c, was in zip(cache[:2], before):
        assert torch.equal(c[0, :, :5], was[0, :, :5]) and (c[0, :, 5] == 0).all() and torch.equal(c[0, :, 6:], was[0, :, 6:])
    ops.evict_kv_i8(*cache, torch.rand(1, 2, 16, generator=g), torch.zeros(1, 1).int(), torch.tensor([16]).int(), torch.ones(1, 1).int(), 16, 2)
    assert torch.equal(cache[0][1], cache[0][0]) and torch.equal(cache[1][1], cache[1][0]) and (cache[2][1] == 0).all()
