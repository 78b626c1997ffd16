"""Keys and values in 8 bits with a magnitude for each page and key head: the checks that the kernels' wrappers and the CPU forms share.

A cache is ``k_cache`` and ``v_cache``, int8 ``[blocks, key heads, page, D]``, and ``kv_max``, fp32 ``[blocks, key heads, 2]``: the largest
magnitude of a page's keys and of its values, a bf16 number as they are. A code stands for ``code * (kv_max / 127)``. The magnitude of a page
grows with what is written behind its first tokens (the codes that are there are rounded again) and begins anew with its first token. A page
that was given a number that is not finite has NaN there, and gives NaN to whoever sees one of its tokens: among the keys to outputs and
weights, among the values to outputs alone.
"""

from __future__ import annotations

from typing import Optional

import torch

from .mx4 import _share_memory, refuse

PAGES = (16, 32, 64)
DIMS = (64, 128)
MAX_GROUP = 16                   # query heads for each key head


_I8, _I32, _F32, _BF16 = torch.int8, torch.int32, torch.float32, torch.bfloat16


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_max: torch.Tensor, what: str) -> tuple[int, int, int, int, int]:
    """Blocks, key heads, page, head dim and device number of a cache."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or k_cache.dtype is not _I8 or v_cache.dtype is not _I8:
        refuse(what, f"k_cache and v_cache are int8 [blocks, key heads, page, D], got {k_cache.dtype} {tuple(shape)} and {v_cache.dtype} "
               f"{tuple(v_cache.shape)}")
    N, H, page, D = shape
    if page not in PAGES or D not in DIMS or N < 1 or H < 1:
        refuse(what, f"pages of 16, 32 or 64 tokens and heads of 64 or 128 columns, got {tuple(shape)}")
    if N * H * page >= 1 << 31:
        refuse(what, f"blocks * key heads * page stay below 2^31, got {tuple(shape)}")
    if kv_max.shape != (N, H, 2) or kv_max.dtype is not _F32:
        refuse(what, f"kv_max is fp32 {(N, H, 2)}, got {kv_max.dtype} {tuple(kv_max.shape)}")
    dev = k_cache.get_device()
    if v_cache.get_device() != dev or kv_max.get_device() != dev:
        refuse(what, "the cache's tensors are on different devices")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and kv_max.is_contiguous()):
        refuse(what, "the cache's tensors are contiguous")
    return N, H, page, D, dev


def check_ints(t: torch.Tensor, name: str, shape: tuple, dev: int, what: str) -> None:
    if t.dtype is not _I32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        refuse(what, f"{name} is contiguous int32 {shape} on the cache's device, got {t.dtype} {tuple(t.shape)} on {t.device}")


def check_tables(block_tables: torch.Tensor, B: int, dev: int, what: str, name: str = "block_tables") -> int:
    shape = block_tables.shape
    if len(shape) != 2 or shape[0] != B or shape[1] < 1 or block_tables.dtype is not _I32 or block_tables.get_device() != dev \
            or not block_tables.is_contiguous():
        refuse(what, f"{name} is contiguous int32 [{B}, pages] on the cache's device, got {block_tables.dtype} {tuple(shape)} on "
               f"{block_tables.device}")
    return shape[1]


def check_lens(ctx_lens: torch.Tensor, dev: int, what: str) -> int:
    shape = ctx_lens.shape
    if len(shape) != 1 or ctx_lens.dtype is not _I32 or ctx_lens.get_device() != dev or not ctx_lens.is_contiguous():
        refuse(what, f"ctx_lens is contiguous int32 [sequences] on the cache's device, got {ctx_lens.dtype} {tuple(shape)} on {ctx_lens.device}")
    return shape[0]


def check_rows(x: torch.Tensor, name: str, heads: Optional[int], D: int, dev: int, what: str) -> tuple[int, int]:
    shape = x.shape
    if len(shape) != 3 or shape[2] != D or heads is not None and shape[1] != heads or x.dtype is not _BF16 or x.get_device() != dev:
        refuse(what, f"{name} is bf16 [tokens, {'heads' if heads is None else heads}, {D}] on the cache's device, got {x.dtype} {tuple(shape)} "
               f"on {x.device}")
    return shape[0], shape[1]


def check_weights(weights: torch.Tensor, seq_slots: Optional[torch.Tensor], B: int, Hkv: int, dev: int, what: str) -> tuple[int, int]:
    """Slots of the weights and tokens of a slot."""
    shape = weights.shape
    if len(shape) != 3 or shape[1] != Hkv or shape[2] < 1 or weights.dtype is not _F32 or weights.get_device() != dev \
            or not weights.is_contiguous():
        refuse(what, f"weights are contiguous fp32 [slots, {Hkv}, tokens] on the cache's device, got {weights.dtype} {tuple(shape)} on "
               f"{weights.device}")
    if seq_slots is not None:
        check_ints(seq_slots, "seq_slots", (B,), dev, what)
    elif shape[0] < B:
        refuse(what, f"weights of {shape[0]} slots for {B} sequences")
    return shape[0], shape[2]


def _rows_2d(t: torch.Tensor) -> torch.Tensor:
    return t.as_strided((t.shape[0], t.shape[1] * t.shape[2]), (t.stride(0), 1), t.storage_offset())


def check_attention(what: str, q: torch.Tensor, cache: tuple, block_tables: torch.Tensor, cu_q: Optional[torch.Tensor],
                    ctx_lens: torch.Tensor, scale: float, window: int, sinks: Optional[torch.Tensor], out: Optional[torch.Tensor],
                    weights: Optional[torch.Tensor], seq_slots: Optional[torch.Tensor], max_ctx: int) -> tuple[int, ...]:
    """Checks what the two attentions share; returns blocks, key heads, page, D, queries, query heads, sequences, pages of a table, window,
    longest sequence, slots of the weights and tokens of a slot."""
    N, Hkv, page, D, dev = check_cache(*cache, what)
    T, Hq = check_rows(q, "q", None, D, dev, what)
    if Hq % Hkv or not 0 < Hq // Hkv <= MAX_GROUP:
        refuse(what, f"1 to {MAX_GROUP} query heads for each key head, got {Hq} and {Hkv}")
    B = check_lens(ctx_lens, dev, what)
    MB = check_tables(block_tables, B, dev, what)
    if cu_q is not None:
        check_ints(cu_q, "cu_q", (B + 1,), dev, what)
    elif T != B:
        refuse(what, f"one query for each sequence, got {T} and {B}")
    if not 0 < scale < float("inf"):
        refuse(what, f"scale is positive and finite, got {scale}")
    if window < 0 or max_ctx < 0:
        refuse(what, f"window and max_ctx are not negative, got {window} and {max_ctx}")
    if sinks is not None and (sinks.shape != (Hq,) or sinks.dtype is not _F32 or sinks.get_device() != dev or not sinks.is_contiguous()):
        refuse(what, f"sinks are contiguous fp32 {(Hq,)} on the cache's device, got {sinks.dtype} {tuple(sinks.shape)} on {sinks.device}")
    if out is not None:
        check_rows(out, "out", Hq, D, dev, what)
        if out.shape[0] != T:
            refuse(what, f"out has the rows of q, got {out.shape[0]} and {T}")
        if out.stride(2) != 1 or out.stride(1) != D or out.stride(0) & 7 or out.data_ptr() & 15 or T > 1 and out.stride(0) < Hq * D:
            refuse(what, "out has neighbouring heads and columns, rows that start on 16 bytes and do not overlap")
        if T > 0 and q.stride(2) == 1 and (q.stride(1) == D or Hq == 1) and _share_memory(_rows_2d(q), _rows_2d(out)):
            refuse(what, "out overlaps the queries")
        lo, hi = out.data_ptr(), out.data_ptr() + 2 * ((T - 1) * out.stride(0) + Hq * D)
        for t in (*cache, weights, sinks):
            if T > 0 and t is not None and t.data_ptr() < hi and lo < t.data_ptr() + t.numel() * t.element_size():
                refuse(what, "out overlaps the cache, the weights or the sinks")
    slots, W = (0, 0) if weights is None else check_weights(weights, seq_slots, B, Hkv, dev, what)
    most = MB * page
    if 0 < max_ctx < most:
        most = max_ctx
    if most >= 1 << 30:
        refuse(what, f"sequences stay below 2^30 tokens, got {most}")
    return N, Hkv, page, D, T, Hq, B, MB, min(window, 1 << 30), most, slots, W


def check_store(what: str, k: torch.Tensor, v: torch.Tensor, cache: tuple, block_tables: torch.Tensor, cu_q: torch.Tensor,
                ctx_lens: torch.Tensor, max_q_len: int) -> tuple[int, ...]:
    """Returns blocks, key heads, page, D, tokens, sequences, pages of a table."""
    N, Hkv, page, D, dev = check_cache(*cache, what)
    T, _ = check_rows(k, "k", Hkv, D, dev, what)
    if check_rows(v, "v", Hkv, D, dev, what)[0] != T:
        refuse(what, f"as many rows of k as of v, got {T} and {v.shape[0]}")
    B = check_lens(ctx_lens, dev, what)
    check_ints(cu_q, "cu_q", (B + 1,), dev, what)
    if max_q_len < 0:
        refuse(what, f"max_q_len is not negative, got {max_q_len}")
    return N, Hkv, page, D, T, B, check_tables(block_tables, B, dev, what)


def check_load(what: str, cache: tuple, block_tables: torch.Tensor, cu_k: torch.Tensor, rows: int) -> tuple[int, ...]:
    """Returns blocks, key heads, page, D, sequences, pages of a table."""
    N, Hkv, page, D, dev = check_cache(*cache, what)
    B = max(cu_k.shape[0] - 1, 0) if cu_k.dim() == 1 else 0
    check_ints(cu_k, "cu_k", (B + 1,), dev, what)
    if rows < 0:
        refuse(what, f"rows is not negative, got {rows}")
    return N, Hkv, page, D, B, check_tables(block_tables, B, dev, what)


def check_evict(what: str, cache: tuple, weights: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor, new_tables: torch.Tensor,
                keep: int, recent: int, first: int, seq_slots: Optional[torch.Tensor]) -> tuple[int, ...]:
    """Returns blocks, key heads, page, D, sequences, pages of a table and of a new one, slots of the weights and tokens of a slot."""
    N, Hkv, page, D, dev = check_cache(*cache, what)
    B = check_lens(ctx_lens, dev, what)
    MB = check_tables(block_tables, B, dev, what)
    MN = check_tables(new_tables, B, dev, what, "new_tables")
    slots, W = check_weights(weights, seq_slots, B, Hkv, dev, what)
    if recent < 0 or first < 0 or keep < 1 or first + recent > keep:
        refuse(what, f"keep at least one token, the first and the recent ones among them: got keep {keep}, recent {recent}, first {first}")
    if B > 0 and new_tables.data_ptr() == block_tables.data_ptr():
        refuse(what, "new_tables have pages of their own, not those of block_tables")
    if keep > MN * page:
        refuse(what, f"keep {keep} tokens need more than the {MN} pages of new_tables")
    return N, Hkv, page, D, B, MB, MN, slots, W
