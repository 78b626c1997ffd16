"""What the wrappers of the 8-bit cache's kernels hand to the library, and what the library refuses: no GPU is needed for either."""

import contextlib

import pytest
import torch

from parallax_b200.ops import _lib, cuda as cu

INVALID_ARG = 1


class Recorder:
    """Stands in for the kernel library: remembers every call, launches nothing."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 256 if name.endswith("_workspace") else 0

        return call


@pytest.fixture
def record(monkeypatch):
    lib = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(cu, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(cu, "_stream", lambda device: 0)
    monkeypatch.setattr(cu, "status_tensor", lambda device: torch.zeros(1, dtype=torch.int32))
    return lib


def _cache():
    return torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2, 2)


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_rows_that_kernels_read_in_vectors(record):
    """Rows keep their stride where they start on 16 bytes and do not overlap; others are copied."""
    flat = torch.randn(4000).bfloat16()
    tab, lens, ends = torch.zeros(3, 1, dtype=torch.int32), _i32(5, 5, 5), _i32(0, 1, 2, 3)
    fine = flat.as_strided((3, 2, 64), (392, 64, 1), 8)
    for q, kept in ((fine, True), (flat.as_strided((3, 2, 64), (392, 64, 1), 1), False), (flat.as_strided((3, 2, 64), (393, 64, 1), 0), False),
                    (flat.as_strided((3, 2, 64), (64, 64, 1), 0), False), (flat.as_strided((3, 2, 64), (392, 72, 1), 0), False),
                    (flat.as_strided((3, 2, 64), (392, 128, 2), 0), False)):
        record.calls.clear()
        cu.attn_decode_i8(q, *_cache(), tab, lens, 0.1)
        cu.attn_prefill_i8(q, *_cache(), tab, ends, lens, 1, 0.1)
        cu.store_kv_i8(q, q, *_cache(), tab, ends, lens, 1)
        calls = {n: a for n, a in record.calls}
        for name, stride in (("pxl_attn_i8_decode", 1), ("pxl_attn_i8_prefill", 1), ("pxl_kv_i8_store", 2)):
            assert (calls[name][0] == q.data_ptr()) == kept and calls[name][stride] == (q.stride(0) if kept else 128)


def test_windows_and_lengths_that_reach_the_library(record):
    q, tab, lens = torch.zeros(1, 2, 64).bfloat16(), torch.zeros(1, 3, dtype=torch.int32), _i32(5)
    for window, want in ((0, 0), (7, 7), (1 << 40, 1 << 30)):
        for max_ctx, longest in ((0, 48), (20, 20), (1000, 48)):
            record.calls.clear()
            cu.attn_decode_i8(q, *_cache(), tab, lens, 0.1, window=window, max_ctx=max_ctx)
            args = dict(record.calls)["pxl_attn_i8_decode"]
            assert args[-4:-2] == (want, longest)


def test_calls_without_work_reach_nothing(record):
    none, tab, lens = torch.zeros(0, 2, 64).bfloat16(), torch.zeros(0, 1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    assert cu.attn_decode_i8(none, *_cache(), tab, lens, 0.1).shape == none.shape
    assert cu.attn_prefill_i8(none, *_cache(), tab, _i32(0), lens, 0, 0.1).shape == none.shape
    cu.store_kv_i8(none, none, *_cache(), tab, _i32(0), lens, 0)
    assert cu.load_kv_i8(*_cache(), tab, _i32(0), 0)[0].shape == none.shape
    cu.evict_kv_i8(*_cache(), torch.zeros(1, 2, 16), tab, lens, tab.clone(), 4, 1)
    assert not record.calls


def _library():
    if not _lib.available():
        pytest.skip("the kernel library is not built")
    return _lib.lib()


P = 1 << 20        # an address that nothing reads: every call below is refused


@pytest.mark.parametrize("change", [dict(D=96), dict(page=8), dict(page=128), dict(Hq=5), dict(Hq=34), dict(Hkv=0), dict(scale=0.0), dict(scale=-1.0),
                                    dict(window=-1), dict(window=(1 << 30) + 1), dict(q_stride=100), dict(out_stride=100), dict(q=P + 2),
                                    dict(out=P + 4), dict(k=P + 8), dict(v=P + 8), dict(m=P + 4), dict(blocks=0), dict(blocks=1 << 40),
                                    dict(max_blocks=0), dict(max_ctx=0), dict(max_ctx=1 << 30), dict(ws=0), dict(ws_bytes=8)])
@pytest.mark.parametrize("decode", [True, False])
def test_attention_refused_by_the_library(change, decode):
    a = dict(q=P, q_stride=256, k=P, v=P, m=P, out=P, out_stride=256, ws=P, ws_bytes=1 << 30, Hq=4, Hkv=2, D=64, page=16, max_blocks=2048, blocks=4096,
             scale=0.1, window=0, max_ctx=30000)
    a.update(change)
    lib = _library()
    head = (a["q"], a["q_stride"], a["k"], a["v"], a["m"], P)
    sizes = (a["Hq"], a["Hkv"], a["D"], a["page"], a["max_blocks"], a["blocks"], a["scale"], a["window"], a["max_ctx"], None, None)
    if decode:
        rc = lib.pxl_attn_i8_decode(*head, P, a["out"], a["out_stride"], None, None, 0, 0, None, a["ws"], a["ws_bytes"], 2, *sizes)
    else:
        rc = lib.pxl_attn_i8_prefill(*head, P, P, a["out"], a["out_stride"], None, None, a["ws"], a["ws_bytes"], 2, 1, 2, *sizes)
    assert rc == INVALID_ARG


@pytest.mark.parametrize("change", [dict(D=96), dict(page=8), dict(Hq=5), dict(scale=0.0), dict(q_stride=100), dict(q=P + 2), dict(lse=0),
                                    dict(weights=0), dict(max_ctx=0), dict(ws=0)])
def test_weights_refused_by_the_library(change):
    a = dict(q=P, q_stride=256, lse=P, weights=P, ws=P, Hq=4, D=64, page=16, scale=0.1, max_ctx=100)
    a.update(change)
    rc = _library().pxl_attn_i8_weigh(a["q"], a["q_stride"], P, P, P, P, P, a["lse"], a["weights"], 100, 1, None, a["ws"], 1 << 30, 5000, 1, 5000, a["Hq"],
                                      2, a["D"], a["page"], 8, 8, a["scale"], 0, a["max_ctx"], None, None)
    assert rc == INVALID_ARG


@pytest.mark.parametrize("change", [dict(D=32), dict(page=48), dict(k_stride=4), dict(v_stride=4), dict(k=P + 2), dict(cache=P + 8), dict(max_blocks=0),
                                    dict(blocks=0)])
def test_store_and_load_refused_by_the_library(change):
    a = dict(k=P, k_stride=128, v_stride=128, cache=P, D=64, page=16, max_blocks=4, blocks=4)
    a.update(change)
    lib = _library()
    tail = (2, a["D"], a["page"], a["max_blocks"], a["blocks"], None, None)
    assert lib.pxl_kv_i8_store(a["k"], P, a["k_stride"], a["v_stride"], P, P, P, a["cache"], P, P, 3, 1, 3, *tail) == INVALID_ARG
    if not {"k", "k_stride", "v_stride"} & set(change):
        assert lib.pxl_kv_i8_load(a["cache"], P, P, P, P, P, P, 3, 1, *tail) == INVALID_ARG


@pytest.mark.parametrize("change", [dict(keep=0), dict(keep=33), dict(recent=-1), dict(first=-1), dict(recent=20, first=20), dict(W=0), dict(max_new=0),
                                    dict(D=8), dict(max_blocks=1 << 28)])
def test_evict_refused_by_the_library(change):
    a = dict(D=64, page=16, max_blocks=4, max_new=2, keep=30, recent=2, first=2, W=64)
    a.update(change)
    rc = _library().pxl_kv_i8_evict(P, P, P, P, a["W"], 1, None, P, P, P, P, P, 1, 2, a["D"], a["page"], a["max_blocks"], a["max_new"], 64, a["keep"],
                                    a["recent"], a["first"], None, None)
    assert rc == INVALID_ARG


def test_workspaces_of_sizes_that_have_none():
    lib = _library()
    assert lib.pxl_attn_i8_decode_workspace(0, 4, 2, 64, 100, 0) == 0
    assert lib.pxl_attn_i8_prefill_workspace(0, 1, 1, 4, 2, 64, 100) == 0
    assert lib.pxl_attn_i8_weigh_workspace(1, 1, 4, 2, 100) == 0
    assert lib.pxl_attn_i8_decode_workspace(2, 4, 2, 64, 100, 1) >= lib.pxl_attn_i8_decode_workspace(2, 4, 2, 64, 100, 0) + 2 * 4 * 128 * 4
