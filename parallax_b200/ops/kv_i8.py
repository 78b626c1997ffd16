"""Keys and values in 8 bits with a magnitude for each page and key head: the checks that the kernels' wrappers and the CPU forms share.

A cache is ``k_cache`` and ``v_cache``, int8 ``[blocks, key heads, page, D]``, and ``kv_max``, fp32 ``[blocks, key heads, 2]``: the largest
magnitude of a page's keys and of its values. A code stands for ``code * (kv_max / 127)``. The magnitude of a page grows with what is written
behind its first tokens (the codes that are there are rounded again) and begins anew with its first token. A page that was given a number
that is not finite has NaN there, and gives NaN to whoever sees one of its tokens.
"""

from __future__ import annotations

from typing import Optional

import torch

from .mx4 import _share_memory, refuse

PAGES = (16, 32, 64)
DIMS = (64, 128)
MAX_GROUP = 16                   # query heads for each key head


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_max: torch.Tensor, what: str) -> tuple[int, int, int, int]:
    """Blocks, key heads, page and head dim of a cache."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or k_cache.dtype is not torch.int8 or v_cache.dtype is not torch.int8:
        refuse(what, f"k_cache and v_cache are int8 [blocks, key heads, page, D], got {k_cache.dtype} {tuple(shape)} and {v_cache.dtype} "
               f"{tuple(v_cache.shape)}")
    if shape[2] not in PAGES or shape[3] not in DIMS or shape[0] < 1 or shape[1] < 1:
        refuse(what, f"pages of 16, 32 or 64 tokens and heads of 64 or 128 columns, got {tuple(shape)}")
    if shape[0] * shape[1] * shape[2] >= 1 << 31:
        refuse(what, f"blocks * key heads * page stay below 2^31, got {tuple(shape)}")
    if kv_max.shape != (shape[0], shape[1], 2) or kv_max.dtype is not torch.float32:
        refuse(what, f"kv_max is fp32 {(shape[0], shape[1], 2)}, got {kv_max.dtype} {tuple(kv_max.shape)}")
    dev = k_cache.device
    if v_cache.device != dev or kv_max.device != dev:
        refuse(what, "the cache's tensors are on different devices")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and kv_max.is_contiguous()):
        refuse(what, "the cache's tensors are contiguous")
    if (k_cache.data_ptr() | v_cache.data_ptr()) & 15 or kv_max.data_ptr() & 7:
        refuse(what, "codes start on 16 bytes, kv_max on 8")
    return tuple(shape)


def check_ints(t: torch.Tensor, name: str, shape: tuple, device: torch.device, what: str) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        refuse(what, f"{name} is contiguous int32 {shape} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def check_tables(block_tables: torch.Tensor, B: int, device: torch.device, what: str, name: str = "block_tables") -> int:
    if block_tables.dim() != 2 or block_tables.shape[1] < 1:
        refuse(what, f"{name} is int32 [sequences, pages], got {tuple(block_tables.shape)}")
    check_ints(block_tables, name, (B, block_tables.shape[1]), device, what)
    return block_tables.shape[1]


def check_rows(x: torch.Tensor, name: str, heads: Optional[int], D: int, device: torch.device, what: str) -> None:
    shape = x.shape
    if len(shape) != 3 or shape[2] != D or heads is not None and shape[1] != heads or x.dtype is not torch.bfloat16 or x.device != device:
        refuse(what, f"{name} is bf16 [tokens, {'heads' if heads is None else heads}, {D}] on {device}, got {x.dtype} {tuple(shape)} on {x.device}")


def check_weights(weights: torch.Tensor, seq_slots: Optional[torch.Tensor], B: int, Hkv: int, device: torch.device, what: str) -> None:
    shape = weights.shape
    if len(shape) != 3 or shape[1] != Hkv or shape[2] < 1 or weights.dtype is not torch.float32 or weights.device != device \
            or not weights.is_contiguous():
        refuse(what, f"weights are contiguous fp32 [slots, {Hkv}, tokens] on {device}, got {weights.dtype} {tuple(shape)} on {weights.device}")
    if seq_slots is not None:
        check_ints(seq_slots, "seq_slots", (B,), device, what)
    elif shape[0] < B:
        refuse(what, f"weights of {shape[0]} slots for {B} sequences")


def _rows_2d(t: torch.Tensor) -> torch.Tensor:
    return t.as_strided((t.shape[0], t.shape[1] * t.shape[2]), (t.stride(0), 1), t.storage_offset())


def check_attention(what: str, q: torch.Tensor, cache: tuple, block_tables: torch.Tensor, cu_q: Optional[torch.Tensor],
                    ctx_lens: torch.Tensor, scale: float, window: int, sinks: Optional[torch.Tensor], out: Optional[torch.Tensor],
                    weights: Optional[torch.Tensor], seq_slots: Optional[torch.Tensor], max_ctx: int) -> tuple[int, ...]:
    """Checks what the two attentions share; returns blocks, key heads, page, D, sequences, pages of a table, longest sequence."""
    N, Hkv, page, D = check_cache(*cache, what)
    dev = cache[0].device
    check_rows(q, "q", None, D, dev, what)
    T, Hq = q.shape[:2]
    if Hq % Hkv or not 0 < Hq // Hkv <= MAX_GROUP:
        refuse(what, f"1 to {MAX_GROUP} query heads for each key head, got {Hq} and {Hkv}")
    B = ctx_lens.shape[0] if ctx_lens.dim() == 1 else -1
    check_ints(ctx_lens, "ctx_lens", (max(B, 0),), dev, what)
    MB = check_tables(block_tables, B, dev, what)
    if cu_q is not None:
        check_ints(cu_q, "cu_q", (B + 1,), dev, what)
    elif T != B:
        refuse(what, f"one query for each sequence, got {T} and {B}")
    if not 0 < scale < float("inf"):
        refuse(what, f"scale is positive and finite, got {scale}")
    if window < 0 or max_ctx < 0:
        refuse(what, f"window and max_ctx are not negative, got {window} and {max_ctx}")
    if sinks is not None and (sinks.shape != (Hq,) or sinks.dtype is not torch.float32 or sinks.device != dev or not sinks.is_contiguous()):
        refuse(what, f"sinks are contiguous fp32 {(Hq,)} on {dev}, got {sinks.dtype} {tuple(sinks.shape)} on {sinks.device}")
    if out is not None:
        check_rows(out, "out", Hq, D, dev, what)
        if out.shape[0] != T:
            refuse(what, f"out has the rows of q, got {out.shape[0]} and {T}")
        if out.stride(2) != 1 or out.stride(1) != D or out.stride(0) & 7 or out.data_ptr() & 15 or T > 1 and out.stride(0) < Hq * D:
            refuse(what, "out has neighbouring heads and columns, rows that start on 16 bytes and do not overlap")
        if T > 0 and q.stride(2) == 1 and q.stride(1) == D and _share_memory(_rows_2d(q), _rows_2d(out)):
            refuse(what, "out overlaps the queries")
    if weights is not None:
        check_weights(weights, seq_slots, B, Hkv, dev, what)
    return N, Hkv, page, D, B, MB, min(max_ctx, MB * page) if max_ctx else MB * page


def check_store(what: str, k: torch.Tensor, v: torch.Tensor, cache: tuple, block_tables: torch.Tensor, cu_q: torch.Tensor,
                ctx_lens: torch.Tensor, max_q_len: int) -> tuple[int, ...]:
    """Returns blocks, key heads, page, D, sequences, pages of a table."""
    N, Hkv, page, D = check_cache(*cache, what)
    dev = cache[0].device
    check_rows(k, "k", Hkv, D, dev, what)
    check_rows(v, "v", Hkv, D, dev, what)
    if k.shape[0] != v.shape[0]:
        refuse(what, f"as many rows of k as of v, got {k.shape[0]} and {v.shape[0]}")
    B = ctx_lens.shape[0] if ctx_lens.dim() == 1 else -1
    check_ints(ctx_lens, "ctx_lens", (max(B, 0),), dev, what)
    check_ints(cu_q, "cu_q", (B + 1,), dev, what)
    if max_q_len < 0:
        refuse(what, f"max_q_len is not negative, got {max_q_len}")
    return N, Hkv, page, D, B, check_tables(block_tables, B, dev, what)


def check_load(what: str, cache: tuple, block_tables: torch.Tensor, cu_k: torch.Tensor, rows: int) -> tuple[int, ...]:
    """Returns blocks, key heads, page, D, sequences, pages of a table."""
    N, Hkv, page, D = check_cache(*cache, what)
    dev = cache[0].device
    B = cu_k.shape[0] - 1 if cu_k.dim() == 1 else -1
    check_ints(cu_k, "cu_k", (max(B, 0) + 1,), dev, what)
    if rows < 0:
        refuse(what, f"rows is not negative, got {rows}")
    return N, Hkv, page, D, B, check_tables(block_tables, B, dev, what)


def check_evict(what: str, cache: tuple, weights: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor, new_tables: torch.Tensor,
                keep: int, recent: int, first: int, seq_slots: Optional[torch.Tensor]) -> tuple[int, ...]:
    """Returns blocks, key heads, page, D, sequences, pages of a table and of a new one."""
    N, Hkv, page, D = check_cache(*cache, what)
    dev = cache[0].device
    B = ctx_lens.shape[0] if ctx_lens.dim() == 1 else -1
    check_ints(ctx_lens, "ctx_lens", (max(B, 0),), dev, what)
    MB = check_tables(block_tables, B, dev, what)
    MN = check_tables(new_tables, B, dev, what, "new_tables")
    check_weights(weights, seq_slots, B, Hkv, dev, what)
    if recent < 0 or first < 0 or keep < 1 or first + recent > keep:
        refuse(what, f"keep at least one token, the first and the recent ones among them: got keep {keep}, recent {recent}, first {first}")
    if keep > MN * page:
        refuse(what, f"keep {keep} tokens need more than the {MN} pages of new_tables")
    return N, Hkv, page, D, B, MB, MN
