"""What the wrappers of the microscaled 4-bit kernels hand to the library, and what the library refuses: no GPU is needed for either."""

import contextlib
import ctypes
import pathlib
import re

import pytest
import torch

from parallax_b200 import ops
from parallax_b200.ops import _lib, cuda as cu

INVALID_ARG = 1


class Recorder:
    """Stands in for the kernel library: remembers every call, launches nothing. `answers`: what a function returns, or calls."""

    def __init__(self, **answers):
        self.answers, self.calls = answers, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            answer = self.answers.get(name, 0)
            return answer(*args) if callable(answer) else answer

        return call


@pytest.fixture
def record(monkeypatch):
    def start(**answers):
        lib = Recorder(**answers)
        monkeypatch.setattr(_lib, "lib", lambda: lib)
        monkeypatch.setattr(cu, "_on", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(cu, "_stream", lambda device: 0)
        monkeypatch.setattr(cu, "status_tensor", lambda device: torch.zeros(1, dtype=torch.int32))
        return lib

    return start


def _bytes(address, n):
    return torch.frombuffer(bytearray(ctypes.string_at(address, n)), dtype=torch.uint8)


def _weight(rows, K, experts=1):
    g = torch.Generator().manual_seed(rows)
    return ops.Mx4Weight.pack(torch.randint(0, 256, (experts * rows, K // 2), generator=g, dtype=torch.uint8),
                              torch.randint(117, 126, (experts * rows, K // 32), generator=g, dtype=torch.uint8), experts)


@pytest.mark.parametrize("few", [0, 1])
@pytest.mark.parametrize("at", [0, 1, 4, 8])
def test_base_of_experts_on_any_address(record, few, at):
    """The kernel that adds the experts' rows up reads `base` in vectors: it gets one that starts on 16 bytes, with the same values."""
    T, K, I, E = 5, 64, 64, 2
    x, ids, wts = torch.randn(T, K).bfloat16(), torch.zeros(T, 2, dtype=torch.int32), torch.ones(T, 2)
    base = torch.randn(T * K + 8).bfloat16()[at:at + T * K].view(T, K)
    seen = []

    def took(position):
        return lambda *args: seen.append((args[position] % 16, _bytes(args[position], 2 * T * K))) or 0

    record(pxl_moe_mx4_few_takes=few, pxl_moe_align_alone=1, pxl_moe_combine_f32=took(3), pxl_moe_mx4_few=took(10))
    cu.moe_ffn_mx4(x, ids, wts, _weight(2 * I, K, E), _weight(K, I, E), base=base)
    (off, values), = seen
    assert off == 0 and torch.equal(values.view(torch.bfloat16).view(T, K), base)


@pytest.mark.parametrize("which", [0, 3, 4])
def test_sum_of_experts_refuses_odd_addresses(which):
    """Refused by the entry point itself, before any launch."""
    args = [0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 1, 1, 64, 0]
    args[which] += 2
    assert _lib.lib().pxl_moe_combine_f32(*args) == INVALID_ARG


def test_base_of_bf16_experts_on_any_address(record):
    """So it is for the experts in bf16: their sum is read in vectors of eight values."""
    T, K, I, E = 5, 64, 64, 2
    base = torch.randn(T * K + 8).bfloat16()[1:1 + T * K].view(T, K)
    seen = []

    def took(*args):
        seen.append((args[3] % 16, _bytes(args[3], 2 * T * K)))
        return 0

    record(pxl_moe_align_alone=1, pxl_moe_combine=took)
    cu.moe_ffn(torch.randn(T, K).bfloat16(), torch.zeros(T, 2, dtype=torch.int32), torch.ones(T, 2), torch.zeros(E * 2 * I, K).bfloat16(),
               torch.zeros(E * K, I).bfloat16(), E, base=base)
    (off, values), = seen
    assert off == 0 and torch.equal(values.view(torch.bfloat16).view(T, K), base)


@pytest.mark.parametrize("which", [0, 3, 4])
def test_sum_of_bf16_experts_refuses_odd_addresses(which):
    args = [0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 1, 1, 64, 0]
    args[which] += 2
    assert _lib.lib().pxl_moe_combine(*args) == INVALID_ARG


@pytest.mark.parametrize("view", ["odd", "wide", "columns"])
def test_rows_of_bf16_experts_on_any_address(record, view):
    """The experts' rows are gathered in vectors, one row of the tokens behind the other."""
    T, K, I, E = 5, 64, 64, 2
    x = {"odd": torch.randn(T * K + 8).bfloat16()[1:1 + T * K].view(T, K), "wide": torch.randn(T, 3 * K).bfloat16()[:, K:2 * K],
         "columns": torch.randn(K, T).bfloat16().t()}[view]
    seen = []

    def took(*args):
        seen.append((args[0] % 16, _bytes(args[0], 2 * T * K)))
        return 0

    record(pxl_moe_align_alone=1, pxl_moe_gather=took)
    cu.moe_ffn(x, torch.zeros(T, 2, dtype=torch.int32), torch.ones(T, 2), torch.zeros(E * 2 * I, K).bfloat16(), torch.zeros(E * K, I).bfloat16(), E)
    (off, values), = seen
    assert off == 0 and torch.equal(values.view(torch.bfloat16).view(T, K), x)


@pytest.mark.parametrize("which", [0, 3])
def test_gathered_rows_refuse_odd_addresses(which):
    args = [0x10000, 0x20000, 0x30000, 0x40000, 1, 64, 0]
    args[which] += 2
    assert _lib.lib().pxl_moe_gather(*args) == INVALID_ARG


def _spoil(t):
    """A bf16 tensor [2, 64] over the first bytes of `t`."""
    return t.flatten().view(torch.uint8)[:256].view(torch.bfloat16).view(2, 64)


@pytest.mark.parametrize("operand", ["codes", "factors", "bias", "rows"])
def test_results_over_an_operand_of_linear_mx4(operand):
    """A result is written while other blocks still read: over weights, their factors, a bias or the rows it is refused."""
    w, x = _weight(64, 64), torch.randn(2, 64).bfloat16()
    bias = torch.zeros(128).bfloat16()[:64]
    out = {"codes": _spoil(w.data), "factors": _spoil(w.row_scale), "bias": torch.zeros(0), "rows": x}[operand]
    if operand == "bias":
        buf = torch.zeros(2, 64).bfloat16()
        bias, out = buf[1], buf
    kept = w.data.clone(), w.row_scale.clone()
    with pytest.raises(ops.KernelError):
        ops.linear_mx4(x, w, bias, out=out)
    assert torch.equal(w.data, kept[0]) and torch.equal(w.row_scale, kept[1])
    assert ops.linear_mx4(x, w, bias, out=torch.empty(2, 64).bfloat16()).shape == (2, 64)


@pytest.mark.parametrize("operand", ["codes", "scales", "w_codes", "w_scales", "bias"])
def test_results_over_an_operand_of_linear_mx4_rows(operand):
    K = 4096
    g = torch.Generator().manual_seed(0)
    t = {n: torch.randint(100, 120, (r, c), generator=g, dtype=torch.uint8)
         for n, r, c in (("codes", 2, K // 2), ("scales", 2, K // 32), ("w_codes", 64, K // 2), ("w_scales", 64, K // 32))}
    buf = torch.zeros(2, 64).bfloat16()
    bias, out = (buf[1], buf) if operand == "bias" else (None, _spoil(t[operand]))
    kept = {n: v.clone() for n, v in t.items()}
    with pytest.raises(ops.KernelError):
        ops.linear_mx4_rows(*t.values(), bias=bias, out=out)
    assert all(torch.equal(v, kept[n]) for n, v in t.items())
    assert ops.linear_mx4_rows(*t.values(), bias=bias, out=torch.empty(2, 64).bfloat16()).shape == (2, 64)


def test_results_over_rows_whose_columns_lie_apart():
    """Rows of a transposed view are copied for the kernels, so that a result may lie anywhere in what they span."""
    w, buf = _weight(64, 64), torch.randn(64, 200).bfloat16()
    x = buf[:, :2].t()
    want = ops.linear_mx4(x.clone(), w)
    for at in (lambda b: b[40:42, 100:164], lambda b: b[:2, :64]):
        b = buf.clone()
        assert torch.equal(ops.linear_mx4(b[:, :2].t(), w, out=at(b)), want)


def test_a_single_row_in_the_place_of_its_residual():
    """The strides of a single row say nothing: the residual may be out, as it may with many."""
    w, x = _weight(64, 64), torch.randn(1, 64).bfloat16()
    buf = torch.randn(1, 128).bfloat16()
    want = ops.linear_mx4(x, w, residual=buf[:, :64].clone())
    for residual, out in ((buf[:1, :64], buf.view(-1)[:64].view(1, 64)), (buf.view(-1)[:64].view(1, 64), buf[:1, :64])):
        kept = buf.clone()
        assert torch.equal(ops.linear_mx4(x, w, residual=residual, out=out), want)
        assert torch.equal(buf[:, :64], want) and torch.equal(buf[:, 64:], kept[:, 64:])
        buf.copy_(kept)
    with pytest.raises(ops.KernelError):
        ops.linear_mx4(x, w, residual=buf[:, 1:65], out=buf[:, :64])
    r = torch.randn(1, 1).bfloat16()
    assert ops.linear_mx4(x, _weight(1, 64), residual=r, out=r) is r


@pytest.mark.parametrize("lo,hi", [(-1, 1), (1, 1), (2, 1), (0, 4), (3, 4), (-2, -1)])
def test_experts_that_a_weight_does_not_have(lo, hi):
    """A slice past the last expert would say that it has experts whose bytes are not its own."""
    w = _weight(64, 64, 3)
    with pytest.raises(ops.KernelError):
        w.expert_slice(lo, hi)
    assert w.expert_slice(1, 3).experts == 2 and w.expert_slice(0, 3).data.numel() == w.data.numel()


def test_weights_of_other_sizes_than_they_say():
    """The kernels take addresses from a weight's sizes: its tensors have to hold that many bytes."""
    w = _weight(130, 160, 2)
    new = ops.Mx4Weight
    assert new(w.data, w.row_scale, 130, 160, 2).cols == 160 and new(w.data, w.row_scale, 256, 256, 2).rows == 256
    odd = torch.zeros(w.data.numel() + 1, dtype=torch.uint8)[1:]
    for args in ((w.data[:-1], w.row_scale, 130, 160, 2), (w.data, w.row_scale, 130, 160, 3), (w.data, w.row_scale, 257, 160, 2),
                 (w.data, w.row_scale, 130, 288, 2), (w.data, w.row_scale, 130, 170, 2), (w.data, w.row_scale[:1], 130, 160, 2),
                 (w.data, w.row_scale.double(), 130, 160, 2), (w.data.int(), w.row_scale, 130, 160, 2), (odd, w.row_scale, 130, 160, 2),
                 (w.data, w.row_scale.t().contiguous().t(), 130, 160, 2), (w.data, w.row_scale, 0, 160, 2), (w.data, w.row_scale, 130, 0, 2),
                 (w.data[:0], w.row_scale[:0], 130, 160, 0), (w.data.to("meta"), w.row_scale, 130, 160, 2)):
        with pytest.raises(ops.KernelError):
            new(*args)


def test_every_entry_point_is_called():
    """What the library exports for microscaled numbers is what the wrappers call."""
    header = (pathlib.Path(_lib.__file__).parents[2] / "csrc" / "pxl_api.h").read_text()
    names = set(re.findall(r"\b(pxl_\w*mx4\w*)\(", header))
    wrappers = pathlib.Path(cu.__file__).read_text()
    assert {"pxl_gemm_mx4", "pxl_moe_mx4_few", "pxl_mx4_pack"} <= names <= set(_lib._SIGS)
    assert all(f".{n}(" in wrappers for n in names)


def test_what_a_laid_out_weight_gives_back():
    """All of a row whose scales are powers within 2^128 of its largest; elsewhere the values that products see, as the docstring says."""
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (4, 48), generator=g, dtype=torch.uint8)
    scales = torch.tensor([[130, 200, 254], [10, 200, 72], [255, 200, 130], [255, 1, 128]], dtype=torch.uint8)
    w = ops.Mx4Weight.pack(codes, scales)
    c, s = w.unpack()
    assert torch.equal(c[0], codes[0]) and torch.equal(s[0], scales[0])
    assert s[1].tolist() == [72, 200, 72] and int(c[1, :16].max()) == 0 and torch.equal(c[1, 16:], codes[1, 16:])   # 10 is below 200 - 128
    assert s[2].tolist() == [255, 128, 58] and torch.isnan(w.row_scale[0, 2])                 # relative to 200, which the factor does not say
    assert torch.equal(s[3], scales[3]) and torch.equal(c[2:], codes[2:])
    assert "NaN" in ops.Mx4Weight.unpack.__doc__ and "mx4.cuh" in ops.Mx4Weight.__doc__
