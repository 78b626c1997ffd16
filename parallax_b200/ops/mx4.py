"""Microscaled 4-bit matrices: the weights' layout, and the checks that the kernels' wrappers and the CPU forms share.

A microscaled matrix ``[rows, K]`` (K a multiple of 32) is held as ``codes`` uint8 ``[rows, K / 2]``, two e2m1 numbers per byte with
the first in the low half, and ``scales`` uint8 ``[rows, K / 32]``, a power of two (e8m0, bias 127, 255 for NaN) per 32 values of a
row: the format of GPT-OSS's ``*_blocks`` (flattened) and ``*_scales``, which the reference hands to its GPU backends untouched
(``src/parallax/sglang/model_runner.py:358-366``).
"""

from __future__ import annotations

from typing import Optional

import torch

from ._lib import EPI_CLIP_GLU, EPI_NONE, EPI_RESIDUAL, EPI_SILU_MUL, KernelError

TILE = 128                       # rows and columns of a block of the layout
CODE_BYTES = TILE * TILE // 2
BLOCK_BYTES = CODE_BYTES + TILE * 4
_SLOTS = ((15, 8, 7, 6), (12, 5, 4, 3), (9, 2, 1, 0), (14, 11, 10, 13))     # bits of sign, two of exponent, mantissa in a half word
_CHUNK = 1 << 24                 # values that are laid out at a time


def refuse(what: str, why: str):
    raise KernelError(f"{what}: {why}")


def check_codes(codes: torch.Tensor, scales: torch.Tensor, what: str) -> tuple[int, int]:
    """Rows and columns of a microscaled matrix."""
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        refuse(what, "codes and scales are uint8 tensors")
    c, s = codes.shape, scales.shape
    if len(c) != 2 or len(s) != 2 or c[0] != s[0] or c[1] != 16 * s[1] or s[1] <= 0:
        refuse(what, f"codes [rows, K / 2] {tuple(c)} need scales [rows, K / 32] {tuple(s)}")
    if codes.device != scales.device:
        refuse(what, "codes and scales are on different devices")
    return c[0], 2 * c[1]


class Mx4Weight:
    """Microscaled weights ``[experts * rows, K]`` as :func:`ops.linear_mx4` and :func:`ops.moe_ffn_mx4` read them, laid out once by
    :meth:`pack`.

    ``data``: per expert, blocks of 128 rows x 128 columns, those of a row of blocks one behind the other. A block holds its codes
    ``[column group of 32][row][16 bytes]`` and then a byte of power per ``[row][column group]``; rows and columns are filled up to
    a whole block with zeros. Eight neighbouring codes share a 32-bit word, the even ones in its low half, the odd ones in its high
    half, with their bits where two at a time become bf16 with few instructions (see ``csrc/mx4.cuh``).
    ``row_scale`` fp32 ``[experts, rows filled up]``: factors of the rows, powers of two (1 where no scale of the row exceeds 128; a
    row with a larger one is stored relative to it, and values 2^128 times smaller than the row's largest scale become 0), NaN where
    the row has a scale of 255."""

    __slots__ = ("data", "row_scale", "rows", "cols", "experts")

    def __init__(self, data: torch.Tensor, row_scale: torch.Tensor, rows: int, cols: int, experts: int = 1):
        # (the kernels take addresses from these sizes)
        nt, kt = -(-rows // TILE), -(-cols // TILE)
        if rows <= 0 or cols <= 0 or cols % 32 or experts <= 0:
            refuse("Mx4Weight", f"{experts} x [{rows}, {cols}]: at least one expert and row, columns in 32s")
        if data.dtype is not torch.uint8 or data.shape != (experts * nt * kt * BLOCK_BYTES,) or not data.is_contiguous() or data.data_ptr() & 15:
            refuse("Mx4Weight", f"data is uint8 [{experts * nt * kt * BLOCK_BYTES}] on 16 bytes, got {data.dtype} {tuple(data.shape)}")
        if row_scale.dtype is not torch.float32 or row_scale.shape != (experts, nt * TILE) or not row_scale.is_contiguous():
            refuse("Mx4Weight", f"row_scale is fp32 [{experts}, {nt * TILE}], got {row_scale.dtype} {tuple(row_scale.shape)}")
        if data.device != row_scale.device:
            refuse("Mx4Weight", "data and row_scale are on different devices")
        self.data, self.row_scale, self.rows, self.cols, self.experts = data, row_scale, rows, cols, experts

    @property
    def device(self) -> torch.device:
        return self.data.device

    def tensors(self) -> list[torch.Tensor]:
        return [self.data, self.row_scale]

    def expert_slice(self, lo: int, hi: int) -> "Mx4Weight":
        """Experts ``[lo, hi)``, as views of this weight."""
        if not 0 <= lo < hi <= self.experts:
            refuse("expert_slice", f"experts [{lo}, {hi}) of {self.experts}")
        n = self.data.numel() // self.experts
        return Mx4Weight(self.data[lo * n:hi * n], self.row_scale[lo:hi], self.rows, self.cols, hi - lo)

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor, experts: int = 1) -> "Mx4Weight":
        """``codes [experts * rows, K / 2]``, ``scales [experts * rows, K / 32]`` -> laid out. Gate and up rows of a gated weight come
        in alternating groups of 64 per expert (:func:`ops.interleave_gate_up`)."""
        total, K = check_codes(codes, scales, "Mx4Weight.pack")
        if experts <= 0 or total <= 0 or total % experts:
            refuse("Mx4Weight.pack", f"{total} rows do not divide by {experts} experts")
        N = total // experts
        dev, nt, kt = codes.device, -(-N // TILE), -(-K // TILE)
        data = torch.empty(experts * nt * kt * BLOCK_BYTES, dtype=torch.uint8, device=dev)
        row_scale = torch.ones((experts, nt * TILE), dtype=torch.float32, device=dev)
        if codes.is_cuda:
            from . import cuda

            cuda.pack_mx4(codes, scales, data, row_scale, experts, N, K)
            return cls(data, row_scale, N, K, experts)
        blocks = data.view(experts, nt, kt, BLOCK_BYTES)
        codes, scales = codes.reshape(experts, N, K // 2), scales.reshape(experts, N, K // 32)
        step = max(1, _CHUNK // (kt * TILE * TILE))
        for e in range(experts):
            for t0 in range(0, nt, step):
                t1 = min(nt, t0 + step)
                n = min(N, t1 * TILE) - t0 * TILE
                pad = torch.nn.functional.pad
                c = pad(codes[e, t0 * TILE:t0 * TILE + n], (0, kt * 64 - K // 2, 0, (t1 - t0) * TILE - n))
                s = pad(scales[e, t0 * TILE:t0 * TILE + n], (0, kt * 4 - K // 32, 0, (t1 - t0) * TILE - n)).int()
                nan = s == 255
                over = (torch.where(nan, torch.zeros_like(s), s).amax(-1) - 128).clamp_min(0)
                row_scale[e, t0 * TILE:t1 * TILE] = torch.where(nan.any(-1), torch.full_like(over, float("nan"), dtype=torch.float32),
                                                                 torch.exp2(over.float()))
                rel = s - over[:, None]
                power = torch.where(nan, torch.full_like(s, 255), rel.clamp_min(0) + 126).to(torch.uint8)
                halves = torch.stack([c & 15, c >> 4], -1).view(-1, kt * 4, 32)
                halves = torch.where((rel < 0)[..., None], torch.zeros_like(halves), halves)
                v = halves.view(t1 - t0, TILE, kt, 4, 4, 4, 2).int()       # [.., block, group, word, slot, half]
                word = torch.zeros(v.shape[:-2] + (2,), dtype=torch.int32, device=dev)
                for i, bits in enumerate(_SLOTS):
                    for j, b in enumerate(bits):
                        word |= ((v[..., i, :] >> (3 - j)) & 1) << b
                by = torch.stack([word & 255, word >> 8], -1).to(torch.uint8)                  # [.., block, group, word, half, byte]
                out = blocks[e, t0:t1]
                out[..., :CODE_BYTES] = by.reshape(t1 - t0, TILE, kt, 4, 16).permute(0, 2, 3, 1, 4).reshape(t1 - t0, kt, CODE_BYTES)
                out[..., CODE_BYTES:] = power.view(t1 - t0, TILE, kt, 4).permute(0, 2, 1, 3).reshape(t1 - t0, kt, TILE * 4)
        return cls(data, row_scale, N, K, experts)

    def unpack(self) -> tuple[torch.Tensor, torch.Tensor]:
        """Codes and scales ``[experts * rows, ...]`` of the values that products see: those that :meth:`pack` was given, but for groups more
        than 2^128 below the largest scale of their row, which come back as zeros with the smallest power that the row holds, and rows with a scale
        of 255, whose other scales come back relative to the largest of them where that exceeds 128 (every result of such a row is NaN)."""
        E, N, K = self.experts, self.rows, self.cols
        nt, kt = -(-N // TILE), -(-K // TILE)
        blocks = self.data.view(E, nt, kt, BLOCK_BYTES)
        by = blocks[..., :CODE_BYTES].reshape(E, nt, kt, 4, TILE, 4, 2, 2).int()               # [.., group, row, word, half, byte]
        word = by[..., 0] | (by[..., 1] << 8)
        v = torch.stack([sum(((word >> b) & 1) << (3 - j) for j, b in enumerate(bits)) for bits in _SLOTS], -2)   # [.., word, slot, half]
        c = (v[..., 0] | (v[..., 1] << 4)).to(torch.uint8).reshape(E, nt, kt, 4, TILE, 16)
        c = c.permute(0, 1, 4, 2, 3, 5).reshape(E, nt * TILE, kt * 64)[:, :N, :K // 2]
        power = blocks[..., CODE_BYTES:].reshape(E, nt, kt, TILE, 4).permute(0, 1, 3, 2, 4).reshape(E, nt * TILE, kt * 4)
        over = torch.log2(torch.nan_to_num(self.row_scale, nan=1.0)).int()[..., None]
        s = torch.where(power == 255, torch.full_like(power, 255).int(), power.int() - 126 + over)[:, :N, :K // 32]
        return c.reshape(E * N, K // 2).contiguous(), s.to(torch.uint8).reshape(E * N, K // 32).contiguous()


def check_rows(x: torch.Tensor, what: str) -> tuple[int, int]:
    shape = x.shape
    if len(shape) != 2 or shape[1] <= 0 or shape[1] % 32:
        refuse(what, f"rows [T, K] with K a multiple of 32, got {tuple(shape)}")
    if x.dtype is not torch.bfloat16 and x.dtype is not torch.float32:
        refuse(what, f"rows are bf16 or fp32, got {x.dtype}")
    return shape[0], shape[1]


def check_weight(w, device: torch.device, what: str) -> None:
    if not isinstance(w, Mx4Weight) or w.experts != 1 or w.data.device != device:
        refuse(what, "w is an Mx4Weight of one expert on the rows' device")


def _check_operand(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype, device: torch.device, what: str) -> None:
    if t.shape != shape or t.dtype is not dtype or t.device != device or t.stride(-1) != 1:
        refuse(what, f"{name} is {dtype} {shape} on {device} with neighbouring columns, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices with neighbouring columns have a byte in common (for rows of unlike strides: may have one)."""
    a0, b0, wa, wb = a.data_ptr(), b.data_ptr(), a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
    sa, sb = a.stride(0) * a.element_size(), b.stride(0) * b.element_size()
    if a0 >= b0 + (b.shape[0] - 1) * sb + wb or b0 >= a0 + (a.shape[0] - 1) * sa + wa:
        return False
    apart = (b0 - a0) % sa if sa == sb and sa > 0 else 0       # columns of one buffer: b's behind a's, and before a's of the next row
    return not (apart >= wa and apart + wb <= sa)


def check_product(what: str, operands: tuple, T: int, N: int, K: int, K_w: int, bias: Optional[torch.Tensor],
                  residual: Optional[torch.Tensor], epi: int, limit: float, out: Optional[torch.Tensor], dtype: torch.dtype) -> int:
    """Checks what the two products share; returns the number of output columns. ``operands``: what is multiplied, the rows first."""
    device = operands[0].device
    if K != K_w:
        refuse(what, f"rows of {K} columns and weights of {K_w}")
    n_out = N
    if epi == EPI_SILU_MUL or epi == EPI_CLIP_GLU:
        n_out = N // 2
        if N % TILE:
            refuse(what, f"a gated product needs gate and up rows in groups of 64, got {N} rows")
        if epi == EPI_CLIP_GLU and not limit > 0:
            refuse(what, "a clipped gate needs limit > 0")
        if residual is not None:
            refuse(what, "a gated product has no residual")
    elif epi == EPI_RESIDUAL:
        if residual is None:
            refuse(what, "EPI_RESIDUAL needs a residual")
    elif epi != EPI_NONE:
        refuse(what, f"unknown epilogue {epi}")
    if bias is not None:
        _check_operand(bias, "bias", (N,), dtype, device, what)
    if residual is not None:
        _check_operand(residual, "residual", (T, n_out), dtype, device, what)
    if out is not None:
        _check_operand(out, "out", (T, n_out), dtype, device, what)
        if T > 1 and out.stride(0) < n_out:
            refuse(what, "rows of out overlap")
        if T > 0 and n_out > 0:
            for t in operands if bias is None else operands + (bias,):
                # (a matrix whose columns lie apart is copied before the kernel runs)
                if (t.stride(-1) == 1 or t.shape[-1] == 1) and _share_memory(t if t.dim() == 2 else t.unsqueeze(0), out):
                    refuse(what, "out overlaps the rows, the weights or the bias")
            # (the residual may be out itself: a result is written by the thread that has read its place)
            if residual is not None and _share_memory(residual, out) and (
                    residual.data_ptr() != out.data_ptr() or T > 1 and residual.stride(0) != out.stride(0)):
                refuse(what, "out overlaps the residual in other places than its own")
    return n_out


def check_experts(what: str, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, w1: Mx4Weight, w2: Mx4Weight,
                  base: Optional[torch.Tensor], act_mode: int, limit: float, b1: Optional[torch.Tensor],
                  b2: Optional[torch.Tensor]) -> None:
    T, K = check_rows(x, what)
    dev = x.device
    shape = ids.shape
    if len(shape) != 2 or shape[0] != T or shape[1] <= 0 or ids.dtype is not torch.int32 or not ids.is_contiguous() or ids.device != dev:
        refuse(what, "ids are int32 [T, k]")
    if weights.shape != shape or weights.dtype is not torch.float32 or not weights.is_contiguous() or weights.device != dev:
        refuse(what, "weights are fp32 of the shape of ids")
    if not isinstance(w1, Mx4Weight) or not isinstance(w2, Mx4Weight) or w1.experts != w2.experts or w1.data.device != dev \
            or w2.data.device != dev:
        refuse(what, "w1 and w2 are Mx4Weights of the same experts on the rows' device")
    if w1.experts > 1024:
        refuse(what, f"{w1.experts} experts, at most 1024")
    if w1.cols != K or w1.rows != 2 * w2.cols or w2.rows != K or w1.rows % TILE:
        refuse(what, f"w1 [2 I, K] and w2 [K, I] with I a multiple of 64, got [{w1.rows}, {w1.cols}] and [{w2.rows}, {w2.cols}] for "
               f"rows of {K}")
    if act_mode != 0 and act_mode != 1:
        refuse(what, "act_mode is 0 (SiLU) or 1 (clipped GLU)")
    if act_mode == 1 and not limit > 0:
        refuse(what, "a clipped gate needs limit > 0")
    for t, name, n in ((b1, "b1", w1.rows), (b2, "b2", w2.rows)):
        if t is not None and (t.numel() != n * w1.experts or not t.is_contiguous() or t.dtype is not x.dtype or t.device != dev):
            refuse(what, f"{name} is {x.dtype} [{w1.experts} * {n}]")
    if base is not None and (base.shape != x.shape or base.dtype is not x.dtype or base.device != dev or not base.is_contiguous()):
        refuse(what, "base has the rows' shape and type")
