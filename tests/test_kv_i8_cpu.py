"""Keys and values in 8 bits on the CPU: the definitions, from differences and in 64 bits, and what the operators refuse."""

import math

import pytest
import torch

from parallax_b200 import ops
from parallax_b200.ops import KernelError
from tests.helpers import kv_i8_oracle as oracle


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cu(new):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)


@pytest.mark.parametrize("page,D", [(16, 64), (32, 128), (64, 64)])
def test_store_then_load_is_off_by_half_a_step(page, D):
    g = _gen(1)
    ctx, new = [page + 3, 2 * page, 1, 5], [page + 3, 7, 1, 0]
    kc, vc, m = oracle.make_cache(g, 12, 3, page, D)
    tables = oracle.tables_for(g, ctx, page, 12)
    k, v = (torch.randn(sum(new), 3, D, generator=g).bfloat16() for _ in range(2))
    before = oracle.values((kc, vc, m), tables[1], ctx[1])
    m_before = m.clone()
    ops.store_kv_i8(k, v, kc, vc, m, tables, _cu(new), torch.tensor(ctx, dtype=torch.int32), max(new))
    got = ops.load_kv_i8(kc, vc, m, tables, _cu(ctx), sum(ctx))
    row, at = 0, 0
    for b, (n, t) in enumerate(zip(new, ctx)):
        for j, x in enumerate((k, v)):
            top = m[tables[b].long()[torch.arange(t) // page]][..., j]                   # [tokens, heads]
            y, step = got[j][at:at + t].double(), top.double()[..., None] / 254          # half a step of a code
            want = x[row:row + n].double()
            assert ((y[t - n:] - want).abs() <= step[t - n:] * (1 + 1e-6) + 2.0 ** -8 * y[t - n:].abs()).all()
            if b == 1:      # tokens that were there: half a step of the new magnitude more, none where it stayed
                old = before[j][:t - n]
                stayed = (m_before[tables[b].long()[torch.arange(t - n) // page]][..., j] == top[:t - n])[..., None]
                far = (y[:t - n] - old).abs() - 2.0 ** -8 * old.abs()
                assert (far <= torch.where(stayed, 1e-6 * old.abs(), step[:t - n] * (1 + 1e-6) + 2.0 ** -16 * old.abs())).all()
        row, at = row + n, at + t


def test_codes_round_ties_to_even_and_magnitudes_begin_anew():
    kc, vc = torch.full((1, 1, 16, 64), 99, dtype=torch.int8), torch.full((1, 1, 16, 64), 99, dtype=torch.int8)
    m = torch.full((1, 1, 2), 1000.0)
    x = torch.zeros(1, 1, 64)
    x[0, 0, :6] = torch.tensor([4.0, 2.0, -2.0, 1.0, -4.0, 0.0])
    ends = torch.tensor([0, 1], dtype=torch.int32)
    tab = torch.zeros(1, 1, dtype=torch.int32)
    ops.store_kv_i8(x.bfloat16(), 0 * x.bfloat16(), kc, vc, m, tab, ends, torch.tensor([1], dtype=torch.int32), 1)
    assert m.flatten().tolist() == [4.0, 0.0]                            # what an earlier owner left does not count
    assert kc[0, 0, 0, :6].tolist() == [127, 64, -64, 32, -127, 0]       # 63.5 -> 64, 31.75 -> 32
    assert (vc[0, 0, 0] == 0).all() and (kc[0, 0, 1:] == 99).all()
    y = torch.zeros(1, 1, 64)
    y[0, 0, 0] = 8.0                                                     # twice the magnitude: 63.5, 32, -32, 16, -63.5 again
    ops.store_kv_i8(y.bfloat16(), y.bfloat16(), kc, vc, m, tab, ends, torch.tensor([2], dtype=torch.int32), 1)
    assert m.flatten().tolist() == [8.0, 8.0]
    assert kc[0, 0, 0, :6].tolist() == [64, 32, -32, 16, -64, 0] and kc[0, 0, 1, 0] == 127 and (kc[0, 0, 2:] == 99).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_number_that_is_not_finite_is_seen_by_those_who_see_the_page(bad):
    g = _gen(2)
    kc, vc, m = oracle.make_cache(g, 4, 2, 16, 64)
    tab = torch.tensor([[0, 1]], dtype=torch.int32)
    x = torch.randn(18, 2, 64, generator=g).bfloat16()
    x[3, 1, 5] = bad
    ops.store_kv_i8(x, x, kc, vc, m, tab, _cu([18]), torch.tensor([18], dtype=torch.int32), 18)
    assert torch.isnan(m[0, 1]).all() and torch.isfinite(m[0, 0]).all() and torch.isfinite(m[1]).all()
    q = torch.randn(1, 4, 64, generator=g).bfloat16()
    full = ops.attn_decode_i8(q, kc, vc, m, tab, torch.tensor([18], dtype=torch.int32), 0.125)
    near = ops.attn_decode_i8(q, kc, vc, m, tab, torch.tensor([18], dtype=torch.int32), 0.125, window=2)
    assert torch.isnan(full[0, 2:]).all() and torch.isfinite(full[0, :2]).all() and torch.isfinite(near).all()
    ops.store_kv_i8(x[:1], x[:1], kc, vc, m, tab, _cu([1]), torch.tensor([1], dtype=torch.int32), 1)
    assert torch.isfinite(m).all()


@pytest.mark.parametrize("window,sink", [(0, False), (5, True), (40, False)])
@pytest.mark.parametrize("decode", [True, False])
def test_attention_and_weights(window, sink, decode):
    g = _gen(3)
    ctx = [37, 1, 20, 0]
    new = [1, 1, 1, 1] if decode else [9, 1, 20, 0]
    cache = oracle.make_cache(g, 6, 2, 16, 64)
    tables = oracle.tables_for(g, ctx, 16, 6)
    q = torch.randn(sum(new), 6, 64, generator=g).bfloat16()
    sinks = torch.randn(6, generator=g) if sink else None
    weights, slots = torch.rand(5, 2, 48, generator=g), torch.tensor([4, 0, 2, 1], dtype=torch.int32)
    before, lens = weights.clone(), torch.tensor(ctx, dtype=torch.int32)
    more = dict(window=window, sinks=sinks, weights=weights, seq_slots=slots)
    if decode:
        out = ops.attn_decode_i8(q, *cache, tables, lens, 0.125, **more)
        assert (out[3] == 0).all()
    else:
        out = ops.attn_prefill_i8(q, *cache, tables, _cu(new), lens, 20, 0.125, **more)
    row = 0
    for b, (o, mean, w, size) in enumerate(oracle.attention(q, cache, tables, new[:3], ctx[:3], 0.125, window, sinks)):
        oracle.assert_output(out[row:row + new[b]], o, mean, size)
        row += new[b]
        want = before[slots[b]].double()
        want[:, :ctx[b]] += w
        oracle.assert_weights(weights[slots[b]], want, before[slots[b]], size, new[b])
        assert (weights[slots[b], :, ctx[b]:] == before[slots[b], :, ctx[b]:]).all()
    assert torch.equal(weights[3], before[3]) and torch.equal(weights[1], before[1])


@pytest.mark.parametrize("keep,recent,first", [(8, 3, 2), (8, 8, 0), (5, 0, 0), (8, 0, 8), (64, 3, 2), (16, 1, 0)])
def test_evict_keeps_the_heaviest(keep, recent, first):
    g = _gen(4)
    ctx = [40, 8, 3, 0, 33]
    cache = oracle.make_cache(g, 40, 2, 16, 64)
    tables = oracle.tables_for(g, ctx, 16, 20)
    new_tables = (torch.randperm(20, generator=g).int() + 20).view(5, 4).contiguous()
    weights = torch.randint(0, 4, (7, 2, 50), generator=g).float()       # many are equal
    weights[3, 0, 11], weights[3, 1, 30], weights[3, 1, 5] = math.nan, -0.0, math.inf
    slots = torch.tensor([3, 0, 6, 1, 2], dtype=torch.int32)
    was, w0 = [oracle.values(cache, tables[b], t) for b, t in enumerate(ctx)], weights.clone()
    kept, lens = ops.evict_kv_i8(*cache, weights, tables, torch.tensor(ctx, dtype=torch.int32), new_tables, keep, recent, first, slots)
    for b, t in enumerate(ctx):
        n = min(t, keep)
        assert int(lens[b]) == n and (kept[b, :, n:] == -1).all()
        now = oracle.values(cache, new_tables[b], n)
        for h in range(2):
            idx = kept[b, h, :n].long()
            row = w0[slots[b], h]
            if t > keep:
                mid = sorted(range(first, t - recent), key=lambda i: (-(math.inf if math.isnan(row[i]) else float(row[i])), not math.isnan(row[i]), i))
                assert idx.tolist() == sorted(list(range(first)) + mid[:keep - first - recent] + list(range(t - recent, t)))
            else:
                assert idx.tolist() == list(range(t))
            w = weights[slots[b], h]
            assert torch.equal(w[:n].nan_to_num(-1), row[idx].nan_to_num(-1)) and (w[n:t] == 0).all() and torch.equal(w[t:], row[t:])
            for j in (0, 1):
                src = cache[2][tables[b].long()[idx // 16], h, j]
                top = torch.stack([src[p - p % 16:p - p % 16 + 16].max() for p in range(n)]) if n else src
                step = torch.where(src == top, 0.0, top.double() / 254)
                assert ((now[j][:, h] - was[b][j][idx, h]).abs() <= step[:, None] * (1 + 1e-12) + 1e-12).all()
    assert torch.equal(weights[4:6], w0[4:6])


def _call(**change):
    g = _gen(5)
    kc, vc, m = oracle.make_cache(g, 4, 2, 16, 64)
    a = dict(q=torch.randn(3, 4, 64, generator=g).bfloat16(), k_cache=kc, v_cache=vc, kv_max=m, block_tables=torch.zeros(3, 1, dtype=torch.int32),
             ctx_lens=torch.ones(3, dtype=torch.int32), scale=0.125)
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    dict(k_cache=torch.zeros(4, 2, 16, 64)), dict(v_cache=torch.zeros(4, 2, 32, 64, dtype=torch.int8)), dict(kv_max=torch.zeros(4, 2)),
    dict(kv_max=torch.zeros(4, 2, 2, dtype=torch.float64)), dict(q=torch.zeros(3, 4, 64)), dict(q=torch.zeros(3, 5, 64).bfloat16()),
    dict(q=torch.zeros(3, 34, 64).bfloat16()), dict(q=torch.zeros(2, 4, 64).bfloat16()), dict(q=torch.zeros(3, 4, 128).bfloat16()),
    dict(block_tables=torch.zeros(3, 1, dtype=torch.int64)), dict(block_tables=torch.zeros(2, 1, dtype=torch.int32)),
    dict(block_tables=torch.zeros(3, 0, dtype=torch.int32)), dict(ctx_lens=torch.ones(3, 1, dtype=torch.int32)), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=math.nan), dict(scale=math.inf), dict(window=-1), dict(max_ctx=-1), dict(sinks=torch.zeros(3)), dict(sinks=torch.zeros(4).double()),
    dict(weights=torch.zeros(3, 3, 16)), dict(weights=torch.zeros(2, 2, 16)), dict(weights=torch.zeros(3, 2, 32)[..., :16]),
    dict(weights=torch.zeros(3, 2, 16), seq_slots=torch.zeros(2, dtype=torch.int32)), dict(out=torch.zeros(3, 4, 64)),
    dict(out=torch.zeros(2, 4, 64).bfloat16()), dict(out=torch.zeros(3, 64, 4).bfloat16().transpose(1, 2)),
    dict(out=torch.zeros(1, 4, 64).bfloat16().expand(3, -1, -1)),
])
def test_attention_refuses(change):
    with pytest.raises(KernelError, match="attn_decode_i8"):
        ops.attn_decode_i8(**_call(**change))


def test_attention_refuses_results_over_queries():
    a = _call()
    with pytest.raises(KernelError, match="overlaps"):
        ops.attn_decode_i8(**a, out=a["q"])
    packed = torch.zeros(3, 8, 64).bfloat16()
    a["q"] = packed[:, :4]
    ops.attn_decode_i8(**a, out=packed[:, 4:])
    for name in ("k_cache", "v_cache", "weights"):
        a = _call(weights=torch.zeros(3, 2, 100))
        over = a[name].flatten().view(torch.uint8)[512:2048].view(torch.bfloat16).view(3, 4, 64)
        with pytest.raises(KernelError, match="overlaps"):
            ops.attn_decode_i8(**a, out=over)
    with pytest.raises(KernelError, match="attn_prefill_i8"):
        b = _call()
        ops.attn_prefill_i8(b["q"], b["k_cache"], b["v_cache"], b["kv_max"], b["block_tables"], torch.zeros(3, dtype=torch.int32), b["ctx_lens"],
                            1, 0.125)


def test_tables_that_are_too_long():
    a = _call(ctx_lens=torch.ones(1, dtype=torch.int32), block_tables=torch.empty(1, (1 << 30) // 16, dtype=torch.int32))
    a["q"] = a["q"][:1]
    with pytest.raises(KernelError, match="2\\^30"):
        ops.attn_decode_i8(**a)


@pytest.mark.parametrize("shape", [(4, 2, 8, 64), (4, 2, 128, 64), (4, 2, 16, 96), (4, 2, 16, 256)])
def test_pages_and_heads_that_are_refused(shape):
    c = torch.zeros(shape, dtype=torch.int8)
    with pytest.raises(KernelError, match="pages of 16, 32 or 64"):
        ops.load_kv_i8(c, c.clone(), torch.zeros(4, 2, 2), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 0)


def test_store_and_evict_refuse():
    g = _gen(6)
    cache = oracle.make_cache(g, 4, 2, 16, 64)
    one, tab = torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 2, 64).bfloat16()
    for k, v, cu, n in ((x.float(), x, _cu([1]), 1), (x, x[:, :1], _cu([1]), 1), (x, torch.cat([x, x]), _cu([1]), 1), (x, x, one, 1),
                        (x, x, _cu([1]), -1)):
        with pytest.raises(KernelError, match="store_kv_i8"):
            ops.store_kv_i8(k, v, *cache, tab, cu, one, n)
    with pytest.raises(KernelError, match="load_kv_i8"):
        ops.load_kv_i8(*cache, tab, _cu([1]), -1)
    w = torch.zeros(1, 2, 16)
    for keep, recent, first, weights, new in ((0, 0, 0, w, tab), (4, 3, 2, w, tab), (17, 1, 0, w, tab), (4, -1, 0, w, tab), (4, 1, -1, w, tab),
                                              (4, 1, 0, w[:, :1], tab), (4, 1, 0, w, torch.zeros(2, 1, dtype=torch.int32))):
        with pytest.raises(KernelError, match="evict_kv_i8"):
            ops.evict_kv_i8(*cache, weights, tab + 0, one, new, keep, recent, first)
    with pytest.raises(KernelError, match="pages of their own"):
        ops.evict_kv_i8(*cache, w, tab, one, tab, 4, 1)


def test_a_prompt_steps_an_eviction_and_more_steps():
    """Against attention over what was written, in 64 bits: the cache's own rounding is in both."""
    g = _gen(7)
    page, D, heads = 16, 64, 2
    cache = [torch.zeros(24, heads, page, D, dtype=torch.int8), torch.zeros(24, heads, page, D, dtype=torch.int8), torch.zeros(24, heads, 2)]
    tab, new_tab = torch.arange(12, dtype=torch.int32).view(2, 6), torch.arange(12, 24, dtype=torch.int32).view(2, 6)
    weights = torch.zeros(2, heads, 96)
    kv = torch.randn(2, 120, 2 * heads, D, generator=g).bfloat16()
    ctx = [50, 41]

    def step(n):
        x = torch.cat([kv[b, c - m:c] for b, (c, m) in enumerate(zip(ctx, n))])
        ends, lens = _cu(n), torch.tensor(ctx, dtype=torch.int32)
        ops.store_kv_i8(x[:, :heads], x[:, heads:], *cache, tab, ends, lens, max(n))
        q = torch.randn(sum(n), 4, D, generator=g).bfloat16()
        if max(n) > 1:
            out = ops.attn_prefill_i8(q, *cache, tab, ends, lens, max(n), 0.125, weights=weights)
        else:
            out = ops.attn_decode_i8(q, *cache, tab, lens, 0.125, weights=weights)
        row = 0
        for b, (o, mean, _, size) in enumerate(oracle.attention(q, cache, tab, n, ctx, 0.125)):
            oracle.assert_output(out[row:row + n[b]], o, mean, size)
            row += n[b]

    step([50, 41])
    for _ in range(3):
        ctx = [c + 1 for c in ctx]
        step([1, 1])
    assert abs(float(weights.sum()) - 4 * (50 + 41 + 6)) < 1e-3          # the weights of a query and head add up to one
    kept, lens = ops.evict_kv_i8(*cache, weights, tab, torch.tensor(ctx, dtype=torch.int32), new_tab, 33, 10, 2)
    assert lens.tolist() == [33, 33] and (kept[:, :, -10:] == torch.tensor(ctx)[:, None, None] - torch.arange(10, 0, -1)).all()
    tab, ctx = new_tab, [33, 33]
    for _ in range(2):
        ctx = [c + 1 for c in ctx]
        step([1, 1])
