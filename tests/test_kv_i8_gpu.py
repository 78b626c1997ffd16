"""The kernels of keys and values in 8 bits: codes, magnitudes and choices as the CPU forms have them, outputs against 64 bits."""

import math

import pytest
import torch

from parallax_b200 import ops
from tests.helpers import kv_i8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cu(new):
    return torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _same(a, b):
    """Equal bit for bit, what is no number at the same places."""
    a, b = a.cpu(), b.cpu()
    return torch.equal(a.nan_to_num(-9, math.inf, -math.inf), b.nan_to_num(-9, math.inf, -math.inf)) if a.is_floating_point() else torch.equal(a, b)


def _check():
    from parallax_b200.ops import cuda as cu

    torch.cuda.synchronize()
    cu.check_status(torch.device(DEV))


# ------------------------------------------------------------------------------------------------ store, load
STORES = [([70, 16, 1, 5, 33], [70, 1, 1, 0, 17]), ([1], [1]), ([300, 129], [300, 100]), ([17, 64, 65, 128], [1, 1, 1, 1])]


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("D,heads", [(64, 3), (128, 2)])
@pytest.mark.parametrize("ctx,new", STORES)
@pytest.mark.parametrize("size", [0.1, 6.0])
def test_store(page, D, heads, ctx, new, size):
    g = _gen(page + D)
    cache = oracle.make_cache(g, 40, heads, page, D)
    tables = oracle.tables_for(g, ctx, page, 40)
    x = (torch.randn(sum(new), 2 * heads + 1, D, generator=g) * size).bfloat16()        # keys and values among other columns
    x[0, 0, 3] = 0
    ends, lens = _cu(new), _i32(ctx)
    dev = _dev(*cache)
    xd = x.to(DEV)
    ops.store_kv_i8(xd[:, 1:heads + 1], xd[:, heads + 1:], *dev, *_dev(tables, ends, lens), max(new))
    ops.store_kv_i8(x[:, 1:heads + 1], x[:, heads + 1:], *cache, tables, ends, lens, max(new))
    _check()
    for a, b in zip(dev, cache):
        assert torch.equal(a.cpu(), b)
    ends = _cu(ctx)
    got = ops.load_kv_i8(*dev, *_dev(tables, ends), sum(ctx) + 3)
    want = ops.load_kv_i8(*cache, tables, ends, sum(ctx) + 3)
    _check()
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_store_of_ties_and_of_very_large_and_small_numbers():
    g = _gen(9)
    heads, D, page = 2, 64, 16
    cache = oracle.make_cache(g, 12, heads, page, D)
    tables = oracle.tables_for(g, [40, 40, 40, 40], page, 12)
    x = torch.randn(4, 40, 2, heads, D, generator=g)
    x[0] = torch.randint(-8, 9, (40, 2, heads, D), generator=g).float()              # halves of the largest
    x[1] *= 1e38
    x[2] *= 1e-39
    x[3, 5:20] = 0
    x = x.bfloat16().flatten(0, 1)
    dev, xd = _dev(*cache), x.to(DEV)
    lens = _i32([40] * 4)
    ops.store_kv_i8(xd[:, 0], xd[:, 1], *dev, *_dev(tables, _cu([40] * 4), lens), 40)
    ops.store_kv_i8(x[:, 0], x[:, 1], *cache, tables, _cu([40] * 4), lens, 40)
    _check()
    for a, b in zip(dev, cache):
        assert _same(a, b)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_store_of_numbers_that_are_not_finite(bad):
    g = _gen(10)
    cache = oracle.make_cache(g, 6, 2, 16, 128)
    tables = oracle.tables_for(g, [20, 30], 16, 6)
    x = torch.randn(12, 2, 2, 128, generator=g).bfloat16()
    x[0, 0, 1, 7] = x[11, 1, 0, 3] = bad
    dev, xd = _dev(*cache), x.to(DEV)
    ops.store_kv_i8(xd[:, 0], xd[:, 1], *dev, *_dev(tables, _cu([2, 10]), _i32([20, 30])), 10)
    ops.store_kv_i8(x[:, 0], x[:, 1], *cache, tables, _cu([2, 10]), _i32([20, 30]), 10)
    _check()
    for a, b in zip(dev, cache):
        assert _same(a, b)


def test_store_of_rows_on_any_address():
    g = _gen(11)
    cache = oracle.make_cache(g, 4, 2, 16, 64)
    tables = oracle.tables_for(g, [20], 16, 4)
    flat = torch.randn(20 * 300 + 8, generator=g).bfloat16()
    views = lambda f: (f[3:].as_strided((20, 2, 64), (300, 65, 1), 3), f.as_strided((20, 2, 64), (300, 128, 2), 1))
    dev = _dev(*cache)
    ops.store_kv_i8(*views(flat.to(DEV)), *dev, *_dev(tables, _cu([20]), _i32([20])), 20)
    ops.store_kv_i8(*views(flat), *cache, tables, _cu([20]), _i32([20]), 20)
    _check()
    for a, b in zip(dev, cache):
        assert torch.equal(a.cpu(), b)


# ------------------------------------------------------------------------------------------------ attention
def _attend(q, cache, tables, new, ctx, scale, window=0, sinks=None, decode=False, weights=None, slots=None, max_ctx=0, out=None):
    d = _dev(*cache, tables, _cu(new), _i32(ctx), sinks, weights, slots)
    more = dict(window=window, sinks=d[6], max_ctx=max_ctx, weights=d[7], seq_slots=d[8])
    if decode:
        out = ops.attn_decode_i8(q, *d[:4], d[5], scale, out=out, **more)
    else:
        out = ops.attn_prefill_i8(q, *d[:4], d[4], d[5], max(new), scale, out=out, **more)
    _check()
    return out.cpu(), None if weights is None else d[7].cpu()


def _compare(seed, new, ctx, G, heads, D, page, window=0, sink=False, decode=False, weighed=False, width=None, mean=0.0):
    g = _gen(seed)
    blocks = sum(-(-t // page) for t in ctx) + 2
    cache = oracle.make_cache(g, blocks, heads, page, D)
    tables = oracle.tables_for(g, ctx, page, blocks, width)
    q = torch.randn(sum(new), G * heads + 2, D, generator=g).bfloat16()          # among other columns of a projection
    sinks = torch.randn(G * heads, generator=g) * 2 if sink else None
    weights = torch.rand(len(ctx) + 2, heads, max(ctx) + 5, generator=g) if weighed else None
    slots = torch.randperm(len(ctx) + 2, generator=g)[:len(ctx)].int() if weighed else None
    scale = D ** -0.5
    out, w = _attend(q.to(DEV)[:, 1:-1], cache, tables, new, ctx, scale, window, sinks, decode, weights, slots, max(ctx))
    row, left = 0, set(range(len(ctx) + 2))
    for b, (o, mean, add, size) in enumerate(oracle.attention(q[:, 1:-1], cache, tables, new, ctx, scale, window, sinks)):
        oracle.assert_output(out[row:row + new[b]], o, mean, size)
        row += new[b]
        if weighed:
            s = int(slots[b])
            left.discard(s)
            want = weights[s].double()
            want[:, :ctx[b]] += add
            oracle.assert_weights(w[s], want, weights[s], size, max(1, new[b]))
    for s in left if weighed else ():
        assert torch.equal(w[s], weights[s])


DECODES = [[1], [65], [2, 16, 17, 63, 64, 128], [777], [5000, 3, 640], [200] * 40]


@pytest.mark.parametrize("ctx", DECODES)
@pytest.mark.parametrize("page,D,G,heads", [(16, 128, 4, 2), (32, 64, 8, 1), (64, 128, 5, 3), (16, 64, 1, 2), (64, 64, 16, 2), (32, 128, 11, 1)])
@pytest.mark.parametrize("weighed", [False, True])
def test_decode(ctx, page, D, G, heads, weighed):
    _compare(sum(ctx) + D, [1] * len(ctx), ctx, G, heads, D, page, decode=True, weighed=weighed)


@pytest.mark.parametrize("window", [1, 16, 100, 1000])
@pytest.mark.parametrize("page,D,G", [(16, 128, 4), (64, 64, 8), (32, 128, 9)])
def test_decode_with_a_window_and_sinks(window, page, D, G):
    _compare(window, [1] * 5, [1, 100, 163, 1024, 15], G, 2, D, page, window=window, sink=True, decode=True, weighed=True)


PROMPTS = [([1], [1]), ([5], [300]), ([128], [128]), ([129, 1, 64], [129, 200, 65]), ([300, 17], [1000, 17]), ([37, 2, 250], [2100, 515, 251])]


@pytest.mark.parametrize("new,ctx", PROMPTS)
@pytest.mark.parametrize("page,D,G,heads", [(16, 128, 4, 2), (32, 64, 8, 1), (64, 128, 5, 2), (16, 64, 1, 2), (64, 64, 16, 1), (32, 128, 11, 1)])
@pytest.mark.parametrize("weighed", [False, True])
def test_prefill(new, ctx, page, D, G, heads, weighed):
    _compare(sum(ctx) + D, new, ctx, G, heads, D, page, weighed=weighed)


@pytest.mark.parametrize("window", [1, 20, 128, 400])
@pytest.mark.parametrize("page,D,G", [(16, 128, 4), (64, 64, 8), (32, 128, 9)])
def test_prefill_with_a_window_and_sinks(window, page, D, G):
    _compare(window, [200, 3, 40], [600, 3, 170], G, 2, D, page, window=window, sink=True, weighed=True)


def test_sequences_without_new_tokens_and_without_any():
    g = _gen(20)
    cache = oracle.make_cache(g, 20, 2, 16, 128)
    tables = oracle.tables_for(g, [30, 40, 0, 50], 16, 20)
    q = torch.randn(23, 8, 128, generator=g).bfloat16()
    out = torch.full((23, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    got, _ = _attend(q.to(DEV), cache, tables, [10, 0, 0, 9], [30, 40, 0, 50], 0.1, out=out)
    want = [x[0] for x in oracle.attention(q[:10], cache, tables[:1], [10], [30], 0.1)] + \
           [x[0] for x in oracle.attention(q[10:19], cache, tables[3:], [9], [50], 0.1)]
    assert (got[:10].double() - want[0]).abs().max() < 0.05 and (got[10:19].double() - want[1]).abs().max() < 0.05
    assert (got[19:] == 7).all()                                         # rows behind the last sequence
    got, _ = _attend(q[:4].to(DEV), cache, tables, [1] * 4, [30, 40, 0, 50], 0.1, decode=True)
    assert (got[2] == 0).all() and got[3].abs().max() > 0
    empty = torch.empty(0, 8, 128, dtype=torch.bfloat16, device=DEV)
    d = _dev(*cache)
    assert ops.attn_decode_i8(empty, *d, torch.empty(0, 4, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV),
                              0.1).shape == (0, 8, 128)


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_what_nobody_sees_is_not_read(decode, D):
    """Magnitudes that are no numbers in pages ahead of the window and behind the context, of keys that some queries do not see."""
    g = _gen(21)
    ctx, new = [200, 70], [1, 1] if decode else [40, 70]
    cache = oracle.make_cache(g, 24, 2, 16, D)
    tables = oracle.tables_for(g, ctx, 16, 24)
    used = set(tables[tables >= 0].tolist())
    for blk in range(24):
        if blk not in used:
            cache[2][blk] = math.nan
    cache[2][int(tables[0, 2])] = math.nan                               # tokens 32 to 47: behind every window
    if not decode:
        cache[2][int(tables[1, 0]), 0, 1] = math.nan                     # values of tokens 0 to 15: for the first 31 queries of a head
    q = torch.randn(sum(new), 8, D, generator=g).bfloat16()
    out, _ = _attend(q.to(DEV), cache, tables, new, ctx, 0.1, window=17, decode=decode)
    row = 0
    for n, (o, mean, _, size) in zip(new, oracle.attention(q, cache, tables, new, ctx, 0.1, 17)):
        oracle.assert_output(out[row:row + n], o, mean, size)
        row += n
    if not decode:
        assert torch.isnan(out[40, 0]).all() and torch.isfinite(out[40, 4:]).all() and torch.isfinite(out[40 + 32:]).all()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_and_values_of_any_size(decode, D):
    """One key far above the others, pages of zeros, magnitudes from 1e-30 to 1e30 side by side, queries of 1e4."""
    g = _gen(22)
    ctx, new = [300], [1] if decode else [70]
    cache = oracle.make_cache(g, 20, 2, 16, D)
    tables = oracle.tables_for(g, ctx, 16, 20)
    t = tables[0].long()
    cache[2][t[0], :, 0] = 60.0
    cache[2][t[3]] = 0.0
    cache[2][t[5], :, 1] = torch.tensor(1e30).bfloat16().float()
    cache[2][t[6], :, 1] = torch.tensor(1e-30).bfloat16().float()
    cache[2][t[7], :, 0] = torch.tensor(1e-30).bfloat16().float()
    q = torch.randn(sum(new), 6, D, generator=g)
    q[:, 1] *= 1e4
    q[:, 2] *= 1e-6
    q = q.bfloat16()
    out, _ = _attend(q.to(DEV), cache, tables, new, ctx, 0.05, decode=decode)
    (o, mean, _, size), = oracle.attention(q, cache, tables, new, ctx, 0.05)
    for h in range(6):                                                   # (each head by its own scores' size)
        (_, _, _, own), = oracle.attention(q[:, h // 3 * 3:h // 3 * 3 + 3][:, h % 3:h % 3 + 1], [c[:, h // 3:h // 3 + 1] for c in cache], tables,
                                           new, ctx, 0.05)
        if 2.0 ** -19 * own < 0.05:
            steps = 300 * 2.0 ** (-35 if decode else -31) * float(cache[2][t, h // 3, 1].max())
            oracle.assert_output(out[:, h], o[:, h], mean[:, h], own, steps)
        else:
            assert torch.isfinite(out[:, h]).all()


@pytest.mark.parametrize("decode", [True, False])
def test_results_in_place_of_other_columns_and_queries_on_any_address(decode):
    g = _gen(23)
    ctx, new = [100, 31], [1, 1] if decode else [50, 31]
    cache = oracle.make_cache(g, 20, 2, 16, 64)
    tables = oracle.tables_for(g, ctx, 16, 20)
    T = sum(new)
    packed = torch.randn(T, 12, 64, generator=g).bfloat16().to(DEV)
    rest = packed[:, 8:].clone()
    q = packed[:, :4].cpu()
    _attend(packed[:, :4], cache, tables, new, ctx, 0.1, decode=decode, out=packed[:, 4:8])
    odd = torch.zeros(T * 300 + 8, dtype=torch.bfloat16, device=DEV)[1:].as_strided((T, 4, 64), (300, 65, 1), 1)
    odd.copy_(q)
    again, _ = _attend(odd, cache, tables, new, ctx, 0.1, decode=decode)
    assert torch.equal(again, packed[:, 4:8].cpu()) and torch.equal(rest, packed[:, 8:])
    row = 0
    for n, (o, mean, _, size) in zip(new, oracle.attention(q, cache, tables, new, ctx, 0.1)):
        oracle.assert_output(again[row:row + n], o, mean, size)
        row += n


@pytest.mark.parametrize("decode", [True, False])
def test_blocks_off_the_cache_and_slots_off_the_weights_are_reported(decode):
    from parallax_b200.ops import cuda as cu

    g = _gen(24)
    cache = _dev(*oracle.make_cache(g, 4, 1, 16, 64))
    q = torch.randn(2, 2, 64, generator=g).bfloat16().to(DEV)
    tab, lens, ends = _dev(_i32([[1, 2], [3, 4]]), _i32([30, 30]), _i32([0, 1, 2]))
    args = (q, *cache, tab, lens, 0.1) if decode else (q, *cache, tab, ends, lens, 1, 0.1)
    run = ops.attn_decode_i8 if decode else ops.attn_prefill_i8
    run(*args)
    with pytest.raises(ops.KernelError, match="block-table"):
        cu.check_status(torch.device(DEV))
    tab.copy_(_i32([[1, 2], [3, -1]]))
    run(*args)
    with pytest.raises(ops.KernelError, match="block-table"):
        cu.check_status(torch.device(DEV))
    tab.copy_(_i32([[1, 2], [3, 0]]))
    weights = torch.zeros(2, 1, 32, device=DEV)
    run(*args, weights=weights, seq_slots=_i32([1, 2]).to(DEV))
    with pytest.raises(ops.KernelError, match="slot"):
        cu.check_status(torch.device(DEV))
    assert abs(float(weights[1].sum()) - 2) < 1e-3 and float(weights[0].sum()) == 0
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device=DEV)
    before = [c.clone() for c in cache]
    ops.store_kv_i8(x, x, *cache, _i32([[1, 4], [1, -1]]).to(DEV), ends, lens, 1)
    with pytest.raises(ops.KernelError, match="slot"):
        cu.check_status(torch.device(DEV))
    assert all(torch.equal(a, b) for a, b in zip(before, cache))


@pytest.mark.parametrize("ends", [[0, 2, 5], [-1, 1, 2], [0, 3, 2]])
def test_ends_off_the_queries(ends):
    """Sequences whose rows are not all there are reported and left out; one that ends before it begins has none."""
    from parallax_b200.ops import cuda as cu

    g = _gen(25)
    cache = _dev(*oracle.make_cache(g, 4, 1, 16, 64))
    q = torch.randn(2, 2, 64, generator=g).bfloat16().to(DEV)
    tab, lens = _dev(_i32([[1, 2], [3, 0]]), _i32([30, 30]))
    out, weights = torch.full((2, 2, 64), 7, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 1, 32, device=DEV)
    ops.attn_prefill_i8(q, *cache, tab, _i32(ends).to(DEV), lens, 1 << 40, 0.1, out=out, weights=weights)
    with pytest.raises(ops.KernelError, match="index"):
        cu.check_status(torch.device(DEV))
    b = 0 if ends == [0, 2, 5] else 1 if ends[0] < 0 else None
    for s in range(2):
        assert abs(float(weights[s].sum()) - (0 if b != s else 2 * (ends[s + 1] - ends[s]))) < 1e-2
    for r in range(2):
        assert bool((out[r] == 7).all()) == (b is None or not ends[b] <= r < ends[b + 1])


def test_evictions_from_one_slot_are_reported():
    """Two sequences with tokens in it; not those without any, as they fill a batch up."""
    from parallax_b200.ops import cuda as cu

    g = _gen(26)
    cache = _dev(*oracle.make_cache(g, 8, 1, 16, 64))
    tab, new = _dev(_i32([[1, 2], [3, 0], [-1, -1]]), _i32([[4], [5], [6]]))
    weights, slots = torch.rand(3, 1, 32, generator=g).to(DEV), _i32([1, 1, 1]).to(DEV)
    run = lambda lens: ops.evict_kv_i8(*cache, weights, tab, _i32(lens).to(DEV), new, 12, 3, seq_slots=slots)
    assert run([0, 30, 0])[1].tolist() == [0, 12, 0]
    _check()
    before = weights.clone()
    kept, lens = run([30, 30, 0])
    with pytest.raises(ops.KernelError, match="slot"):
        cu.check_status(torch.device(DEV))
    assert (kept == -1).all() and (lens == 0).all() and torch.equal(weights, before)


# ------------------------------------------------------------------------------------------------ evict
@pytest.mark.parametrize("page,D", [(16, 128), (32, 64), (64, 128), (16, 64), (64, 64)])
@pytest.mark.parametrize("keep,recent,first", [(64, 20, 4), (64, 64, 0), (33, 0, 0), (40, 0, 40), (300, 7, 1), (1, 0, 0)])
@pytest.mark.parametrize("kind", ["spread", "equal", "odd"])
def test_evict(page, D, keep, recent, first, kind):
    g = _gen(page + keep)
    heads, ctx = 3, [700, 64, 65, 3, 0, 311, 1300]
    pages = -(-keep // page)
    cache = oracle.make_cache(g, 200 + 7 * pages, heads, page, D)
    tables = oracle.tables_for(g, ctx, page, 200)
    new_tables = (torch.randperm(7 * pages, generator=g).int() + 200).view(7, pages).contiguous()
    weights = torch.exp(3 * torch.randn(9, heads, 1400, generator=g))
    if kind == "equal":
        weights = torch.randint(0, 3, (9, heads, 1400), generator=g).float()
    if kind == "odd":
        weights[:, :, ::7], weights[:, :, ::5], weights[:, 1, ::11], weights[:, 2, ::3] = 0.0, -0.0, math.nan, math.inf
        weights[:, 0, 100:200] *= -1
    slots = torch.randperm(9, generator=g)[:7].int()
    d = _dev(*cache, weights, tables, _i32(ctx), new_tables)
    kept, lens = ops.evict_kv_i8(*d, keep, recent, first=first, seq_slots=slots.to(DEV))
    want, want_lens = ops.evict_kv_i8(*cache, weights, tables, _i32(ctx), new_tables, keep, recent, first=first, seq_slots=slots)
    _check()
    assert torch.equal(kept.cpu(), want) and torch.equal(lens.cpu(), want_lens)
    assert torch.equal(d[3].cpu().nan_to_num(-9), weights.nan_to_num(-9))
    for a, b in zip(d[:3], cache):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("n,keep", [(40000, 5000), (70001, 9), (33000, 32000)])
def test_evict_from_long_sequences(n, keep):
    g = _gen(n)
    blocks = -(-n // 16) + -(-keep // 16)
    cache = oracle.make_cache(g, blocks, 1, 16, 64)
    tables, new_tables = torch.arange(-(-n // 16)).int()[None], torch.arange(-(-n // 16), blocks).int()[None]
    weights = torch.rand(1, 1, n, generator=g).mul(5000).round()          # some are equal
    d = _dev(*cache, weights, tables, _i32([n]), new_tables)
    kept, _ = ops.evict_kv_i8(*d, keep, 3, first=2)
    want, _ = ops.evict_kv_i8(*cache, weights, tables, _i32([n]), new_tables, keep, 3, first=2)
    _check()
    assert torch.equal(kept.cpu(), want) and torch.equal(d[3].cpu(), weights) and torch.equal(d[0].cpu(), cache[0])


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("page,D", [(16, 128), (64, 64)])
def test_a_prompt_steps_an_eviction_and_more_steps(page, D):
    """As a server would use them, every step against attention over what was written."""
    g = _gen(30)
    heads, G = 2, 4
    most = -(-400 // page)
    cache = _dev(torch.zeros(4 * most, heads, page, D, dtype=torch.int8), torch.zeros(4 * most, heads, page, D, dtype=torch.int8),
                 torch.full((4 * most, heads, 2), math.nan))
    tab, new_tab = _dev(torch.arange(2 * most).int().view(2, most), (torch.arange(2 * most) + 2 * most).int().view(2, most))
    weights = torch.zeros(2, heads, 400, device=DEV)
    kv = torch.randn(2, 500, 2 * heads, D, generator=g).bfloat16()
    ctx, n_steps = [250, 141], 0

    def step(n):
        x = torch.cat([kv[b, c - m:c] for b, (c, m) in enumerate(zip(ctx, n))]).to(DEV)
        ends, lens = _dev(_cu(n), _i32(ctx))
        q = torch.randn(sum(n), G * heads, D, generator=g).bfloat16()
        ops.store_kv_i8(x[:, :heads], x[:, heads:], *cache, tab, ends, lens, max(n))
        more = dict(weights=weights, max_ctx=max(ctx))
        if max(n) > 1:
            out = ops.attn_prefill_i8(q.to(DEV), *cache, tab, ends, lens, max(n), 0.125, **more)
        else:
            out = ops.attn_decode_i8(q.to(DEV), *cache, tab, lens, 0.125, **more)
        _check()
        row = 0
        for b, (o, mean, _, size) in enumerate(oracle.attention(q, [c.cpu() for c in cache], tab.cpu(), n, ctx, 0.125)):
            oracle.assert_output(out[row:row + n[b]].cpu(), o, mean, size)
            row += n[b]

    step([250, 141])
    for _ in range(4):
        ctx = [c + 1 for c in ctx]
        step([1, 1])
    assert abs(float(weights.sum()) - G * heads * (250 + 141 + 8)) < 0.05
    kept, lens = ops.evict_kv_i8(*cache, weights, tab, _i32(ctx).to(DEV), new_tab, 100, 30, first=4)
    assert lens.tolist() == [100, 100]
    tab, ctx = new_tab, [100, 100]
    for _ in range(3):
        ctx = [c + 1 for c in ctx]
        step([1, 1])


def _case(seed, decode):
    g = _gen(seed)
    ctx = [900, 333, 64]
    new = [1, 1, 1] if decode else [150, 333, 1]
    blocks = sum(-(-t // 16) for t in ctx)
    cache = oracle.make_cache(g, blocks, 2, 16, 128)
    tables = oracle.tables_for(g, ctx, 16, blocks)
    q = torch.randn(sum(new), 8, 128, generator=g).bfloat16()
    d = _dev(q, *cache, tables, _cu(new), _i32(ctx))
    weights = torch.zeros(3, 2, 900, device=DEV)

    def run():
        if decode:
            return ops.attn_decode_i8(*d[:5], d[6], 0.1, weights=weights)
        return ops.attn_prefill_i8(*d[:7], max(new), 0.1, weights=weights)

    return run, d, weights


@pytest.mark.parametrize("decode", [True, False])
def test_the_same_bits_on_every_run(decode):
    run, _, weights = _case(40, decode)
    first = run().clone()
    w = weights.clone()
    for _ in range(5):
        weights.zero_()
        assert torch.equal(run(), first) and torch.equal(weights, w)
    _check()


def test_two_graphs_that_run_side_by_side():
    a, da, wa = _case(41, True)
    b, db, wb = _case(42, False)
    want = [a().clone(), b().clone()]
    weigh = [wa.clone(), wb.clone()]
    graphs, outs = [], []
    for run in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        wa.zero_()
        wb.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want)) and torch.equal(wa, weigh[0]) and torch.equal(wb, weigh[1])
    new_q = torch.randn_like(da[0])
    da[0].copy_(new_q)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], a())
    _check()


def test_store_attention_and_eviction_in_a_launch_chain():
    from parallax_b200.ops import cuda as cu

    g = _gen(50)
    cache = _dev(*oracle.make_cache(g, 60, 2, 16, 128))
    tab, new_tab = _dev(torch.arange(40).int().view(2, 20), (torch.arange(20) + 40).int().view(2, 10))
    x = torch.randn(2, 4, 128, generator=g).bfloat16().to(DEV)
    q = torch.randn(2, 8, 128, generator=g).bfloat16().to(DEV)
    ends, lens = _dev(_i32([0, 1, 2]), _i32([300, 170]))

    def go(cache, weights):
        ops.store_kv_i8(x[:, :2], x[:, 2:], *cache, tab, ends, lens, 1)
        out = ops.attn_decode_i8(q, *cache, tab, lens, 0.1, weights=weights)
        _, n = ops.evict_kv_i8(*cache, weights, tab, lens, new_tab, 150, 10)
        return out, ops.attn_decode_i8(q, *cache, new_tab, n, 0.1), weights, *cache

    want = go([c.clone() for c in cache], torch.zeros(2, 2, 320, device=DEV))
    _check()
    for _ in range(20):
        mine, w = [c.clone() for c in cache], torch.zeros(2, 2, 320, device=DEV)
        with cu.launch_chain():
            got = go(mine, w)
        _check()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ sizes, streams, odd lengths
def test_more_new_tokens_than_tokens():
    """Queries at positions below zero see nothing; the others see the tokens that are there."""
    g = _gen(60)
    cache = oracle.make_cache(g, 4, 1, 16, 64)
    q = torch.randn(9, 2, 64, generator=g).bfloat16()
    d = _dev(q, *cache, _i32([[0], [1]]), _i32([0, 5, 9]), _i32([3, 0]))
    out = torch.full((9, 2, 64), 5.0, dtype=torch.bfloat16, device=DEV)
    weights = torch.zeros(2, 1, 16, device=DEV)
    ops.attn_prefill_i8(*d, 5, 0.1, out=out, weights=weights)
    _check()
    assert (out[:2] == 0).all() and (out[5:] == 0).all()
    (o, mean, add, size), = oracle.attention(q[2:5], cache, _i32([[0]]), [3], [3], 0.1)
    oracle.assert_output(out[2:5].cpu(), o, mean, size)
    oracle.assert_weights(weights[0, :, :3].cpu(), add, torch.zeros(1, 3), size, 3)
    assert (weights[0, :, 3:] == 0).all() and (weights[1] == 0).all()


@pytest.mark.parametrize("page,D", [(64, 128), (16, 64)])
def test_blocks_past_two_and_four_gigabytes(page, D):
    """Offsets above 2^31 and 2^32 bytes in the cache: the same codes and results as at its start."""
    heads, G = 8, 2
    blocks = (9 << 29) // (heads * page * D)
    g = _gen(61)
    k, v = (torch.zeros(blocks, heads, page, D, dtype=torch.int8, device=DEV) for _ in range(2))
    m = torch.zeros(blocks, heads, 2, device=DEV)
    n = 3 * page + 5
    x = torch.randn(n, 2 * heads, D, generator=g).bfloat16().to(DEV)
    q = torch.randn(n, G * heads, D, generator=g).bfloat16().to(DEV)
    ends, lens = _dev(_i32([0, n]), _i32([n]))
    got = []
    for first in (0, blocks // 2 - 2, blocks - 8):
        tab = torch.arange(first, first + 4).int()[None].to(DEV)
        new_tab = torch.arange(first + 4, first + 8).int()[None].to(DEV)
        weights = torch.zeros(1, heads, n, device=DEV)
        ops.store_kv_i8(x[:, :heads], x[:, heads:], k, v, m, tab, ends, lens, n)
        r = [*ops.load_kv_i8(k, v, m, tab, ends, n), ops.attn_prefill_i8(q, k, v, m, tab, ends, lens, n, 0.1, weights=weights),
             ops.attn_decode_i8(q[:1], k, v, m, tab, lens, 0.1, weights=weights)]
        kept, n_kept = ops.evict_kv_i8(k, v, m, weights, tab, lens, new_tab, 2 * page + 1, 7)
        r += [kept, weights, *ops.load_kv_i8(k, v, m, new_tab, _i32([0, 2 * page + 1]).to(DEV), 2 * page + 1)]
        got.append(r)
    _check()
    for r in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, got[0]))


@pytest.mark.parametrize("decode", [True, False])
def test_on_a_stream_of_its_own(decode):
    run, d, weights = _case(62, decode)
    want = run().clone()
    weigh = weights.clone()
    _check()
    s = torch.cuda.Stream()
    q = d[0].clone()
    for _ in range(3):
        with torch.cuda.stream(s):
            d[0].zero_()
            weights.zero_()
            d[0].copy_(q)                 # the inputs come on this stream, right before
            got = run()
        s.synchronize()
        assert torch.equal(got, want) and torch.equal(weights, weigh)
    _check()


@pytest.mark.parametrize("G", [1, 3, 16])
def test_one_long_sequence(G):
    """Many CTAs for a pair, in decoding as for a few new tokens, with sinks and weights."""
    _compare(63 + G, [1], [20011], G, 1, 128, 64, sink=True, decode=True, weighed=True)
    _compare(64 + G, [9], [12007], G, 1, 64, 16, sink=True, weighed=True)


def test_many_short_sequences():
    _compare(65, [1] * 700, [1 + 7 * i % 90 for i in range(700)], 4, 2, 64, 16, decode=True)
    _compare(66, [1 + i % 3 for i in range(300)], [3 + 11 * i % 50 for i in range(300)], 2, 1, 128, 32, weighed=True)


@pytest.mark.parametrize("seqs,heads,most", [(5, 2, 256), (5, 2, 257), (40, 2, 512), (40, 2, 513), (300, 4, 1024), (300, 4, 1025)])
@pytest.mark.parametrize("D,G", [(64, 4), (128, 2), (64, 9)])
def test_sequences_that_are_cut_and_that_are_not(seqs, heads, most, D, G):
    """On both sides of the lengths up to which a (sequence, key head) pair stays in one CTA, lengths of all kinds."""
    g = _gen(67 + seqs + most)
    ctx = [most] + torch.randint(1, most + 1, (seqs - 1,), generator=g).tolist()
    _compare(68 + most, [1] * seqs, ctx, G, heads, D, 16, sink=True, decode=True, weighed=seqs == 40)


@pytest.mark.parametrize("window", [129, 193, 194, 400])
def test_windows_that_are_cut_and_that_are_not(window):
    ctx = [1, 64, 3000, 129, 700, 193, 2047, 385, 2048, 1000]
    _compare(window, [1] * 10, ctx, 8, 2, 64, 32, window=window, sink=True, decode=True, weighed=True)


@pytest.mark.parametrize("seqs,heads,most", [(3, 4, 2048), (24, 4, 1500), (27, 8, 700), (40, 8, 700), (12, 8, 2049), (1, 1, 8193), (2, 2, 9000)])
@pytest.mark.parametrize("D,G,weighed", [(64, 4, True), (128, 5, False), (128, 16, True), (64, 1, False), (64, 12, False)])
def test_pairs_that_ctas_share(seqs, heads, most, D, G, weighed):
    """Eight, four and two CTAs in a cluster for each pair, and pairs that are dealt out to all; some sequences shorter than the CTAs are many."""
    g = _gen(69 + seqs + most)
    ctx = [most] + torch.randint(0, most + 1, (seqs - 1,), generator=g).tolist()
    ctx[-1] = ctx[-1] if seqs < 3 else 100
    _compare(70 + most, [1] * seqs, ctx, G, heads, D, 32, sink=True, decode=True, weighed=weighed)
