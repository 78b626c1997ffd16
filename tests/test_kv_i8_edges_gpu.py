"""The kernels of keys and values in 8 bits where a call is at its edges: pages without a magnitude, sequences that are longer than a call
says, slots that sequences share, magnitudes far apart."""

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


def _check():
    from parallax_b200.ops import cuda as cu

    torch.cuda.synchronize()
    cu.check_status(torch.device(DEV))


def _reported(match):
    """A device status that was set, taken back."""
    from parallax_b200.ops import cuda as cu

    with pytest.raises(ops.KernelError, match=match):
        cu.check_status(torch.device(DEV))


def _attend(q, cache, tables, new, ctx, scale, window=0, sinks=None, weights=None, slots=None, max_ctx=0):
    """Outputs and weights on the CPU; one new token each: the form for single queries."""
    d = _dev(*cache, tables, _i32(ctx), sinks, weights, slots)
    more = dict(window=window, sinks=d[5], max_ctx=max_ctx, weights=d[6], seq_slots=d[7])
    if max(new) == 1:
        out = ops.attn_decode_i8(q.to(DEV), *d[:5], scale, **more)
    else:
        out = ops.attn_prefill_i8(q.to(DEV), *d[:4], _cu(new).to(DEV), d[4], max(new), scale, **more)
    _check()
    return out.cpu(), None if weights is None else d[6].cpu()


# ------------------------------------------------------------------------------------------------ sequences that are reported
@pytest.mark.parametrize("ends", [[0, 2, 5], [-1, 1, 2], [0, 3, 2]])
def test_ends_off_the_queries_of_long_sequences(ends):
    """As with short ones: reported, their rows left as they are; their keys would be split over CTAs."""
    g = _gen(3)
    cache = _dev(*oracle.make_cache(g, 500, 1, 16, 64))
    q = torch.randn(2, 2, 64, generator=g).bfloat16().to(DEV)
    tab, lens = torch.randperm(500, generator=g).int().view(2, 250).to(DEV), _i32([4000, 3900]).to(DEV)
    out, weights = torch.full((2, 2, 64), 7, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 1, 4000, device=DEV)
    ops.attn_prefill_i8(q, *cache, tab, _i32(ends).to(DEV), lens, 1 << 40, 0.1, out=out, weights=weights)
    _reported("index")
    b = 0 if ends == [0, 2, 5] else 1 if ends[0] < 0 else None
    for s in range(2):
        assert abs(float(weights[s].sum()) - (0 if b != s else 2 * (ends[s + 1] - ends[s]))) < 1e-2
    for r in range(2):
        assert bool((out[r] == 7).all()) == (b is None or not ends[b] <= r < ends[b + 1])


# ------------------------------------------------------------------------------------------------ more new tokens than a call says
@pytest.mark.parametrize("ctx", [60, 4000])
@pytest.mark.parametrize("G", [2, 16])
def test_prompts_of_more_new_tokens_than_the_call_says(ctx, G):
    """Reported and left out, by the outputs and by the weights; the sequence beside them is not touched by that. 4000 tokens: keys are
    split over CTAs."""
    g = _gen(1)
    new, D = [40, 3], 64
    blocks = 2 * -(-ctx // 16)
    cache = oracle.make_cache(g, blocks, 1, 16, D)
    tables = oracle.tables_for(g, [ctx, ctx], 16, blocks)
    q = torch.randn(43, G, D, generator=g).bfloat16()
    before = torch.rand(2, 1, ctx, generator=g)
    d = _dev(q, *cache, tables, _cu(new), _i32([ctx, ctx]), before)
    out = torch.full((43, G, D), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.attn_prefill_i8(*d[:7], 39, 0.1, out=out, weights=d[7])
    _reported("index")
    (_, _, _, _), (o, mean, add, size) = oracle.attention(q, cache, tables, new, [ctx, ctx], 0.1)
    assert (out[:40] == 7).all() and torch.equal(d[7][0].cpu(), before[0])
    oracle.assert_output(out[40:].cpu(), o, mean, size)
    oracle.assert_weights(d[7][1].cpu(), before[1].double() + add, before[1], size, 3)
    ops.attn_prefill_i8(*d[:7], 0, 0.1, out=out, weights=d[7])
    _reported("index")
    assert (out[:40] == 7).all()
    ops.attn_prefill_i8(*d[:7], 40, 0.1, out=out)
    _check()
    assert not (out[:40] == 7).all()


@pytest.mark.parametrize("most", [0, 1, 16, 39])
@pytest.mark.parametrize("page", [16, 64])
def test_store_of_more_new_tokens_than_the_call_says(most, page):
    g = _gen(2)
    cache = _dev(*oracle.make_cache(g, 12, 2, page, 64))
    tables = oracle.tables_for(g, [70, 50], page, 12).to(DEV)
    x = torch.randn(40 + most, 4, 64, generator=g).bfloat16().to(DEV)
    want = [c.clone() for c in cache]
    ends, lens = _dev(_i32([0, 40, 40 + most]), _i32([70, 50]))
    if most > 0:
        ops.store_kv_i8(x[40:, :2], x[40:, 2:], *want, tables[1:], _i32([0, most]).to(DEV), lens[1:], most)
    _check()
    ops.store_kv_i8(x[:, :2], x[:, 2:], *cache, tables, ends, lens, most)
    _reported("index")
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


# ------------------------------------------------------------------------------------------------ pages without a magnitude
FORMS = [([1] * 3, [2048, 1500, 31], 4),                  # single queries: a cluster for each pair
         ([1] * 12, [2049] + [300] * 11, 8),              # pairs dealt out
         ([1] * 40, [200] * 40, 2),                       # pairs left whole
         ([300, 17], [1000, 17], 2),                      # prompts
         ([37], [2100], 2)]                               # keys split over CTAs


@pytest.mark.parametrize("new,ctx,heads", FORMS)
@pytest.mark.parametrize("page,D,G", [(16, 128, 4), (64, 64, 9), (32, 64, 1)])
@pytest.mark.parametrize("window", [0, 150])
def test_values_without_a_magnitude_leave_the_weights_as_they_should_be(new, ctx, heads, page, D, G, window):
    """What a token got depends on keys alone: outputs are no numbers for those who see it, weights and the other outputs are right."""
    g = _gen(4)
    blocks = sum(-(-t // page) for t in ctx)
    cache = oracle.make_cache(g, blocks, heads, page, D)
    tables = oracle.tables_for(g, ctx, page, blocks)
    for b, t in enumerate(ctx):                            # a page in the middle of head 0's, the last one of head 1's
        if b % 3 < 2:
            cache[2][int(tables[b, (t - 1) // 2 // page]), 0, 1] = math.nan
            cache[2][int(tables[b, (t - 1) // page]), 1, 1] = math.nan
    q = torch.randn(sum(new), G * heads, D, generator=g).bfloat16()
    weights, scale = torch.rand(len(ctx), heads, max(ctx), generator=g), D ** -0.5
    out, w = _attend(q, cache, tables, new, ctx, scale, window, weights=weights, max_ctx=max(ctx))
    row = 0
    for b, (o, mean, add, size) in enumerate(oracle.attention(q, cache, tables, new, ctx, scale, window)):
        assert torch.isfinite(add).all() and (b % 3 == 2 or torch.isnan(o).any())
        oracle.assert_output(out[row:row + new[b]], o, mean, size)
        want = weights[b].double()
        want[:, :ctx[b]] += add
        oracle.assert_weights(w[b], want, weights[b], size, new[b])
        row += new[b]


@pytest.mark.parametrize("new,ctx,heads", FORMS)
def test_keys_without_a_magnitude(new, ctx, heads):
    """Scores that are no numbers: neither outputs nor weights are numbers for those who see the page, all others are right."""
    g = _gen(5)
    blocks = sum(-(-t // 16) for t in ctx)
    cache = oracle.make_cache(g, blocks, heads, 16, 64)
    tables = oracle.tables_for(g, ctx, 16, blocks)
    cache[2][int(tables[0, ctx[0] // 2 // 16]), 0, 0] = math.nan
    q = torch.randn(sum(new), 4 * heads, 64, generator=g).bfloat16()
    weights = torch.rand(len(ctx), heads, max(ctx), generator=g)
    out, w = _attend(q, cache, tables, new, ctx, 0.125, weights=weights, max_ctx=max(ctx))
    whole = [c.clone() for c in cache]
    whole[2][int(tables[0, ctx[0] // 2 // 16]), 0, 0] = 1.0
    row = 0
    first = ctx[0] // 2 // 16 * 16 - (ctx[0] - new[0])     # the first query of sequence 0 that sees the page
    for b, (o, mean, add, size) in enumerate(oracle.attention(q, whole, tables, new, ctx, 0.125)):
        if b == 0:
            o[max(first, 0):, :4] = math.nan
            assert torch.isnan(w[0, 0, :ctx[0]]).all()
        oracle.assert_output(out[row:row + new[b]], o, mean, size)
        want = weights[b].double()
        want[:, :ctx[b]] += add
        for h in range(heads):
            if b or h:
                oracle.assert_weights(w[b, h], want[h], weights[b, h], size, new[b])
        row += new[b]


# ------------------------------------------------------------------------------------------------ magnitudes far apart
@pytest.mark.parametrize("big", [2.0 ** 30, 1e30, 3e38])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("new,ctx", [(200, 200), (80, 400), (80, 3000)])
@pytest.mark.parametrize("page,D,G", [(16, 128, 4), (64, 64, 1), (32, 64, 16)])
def test_values_that_only_other_queries_see(big, window, new, ctx, page, D, G):
    """A page whose values are far above the others': those who do not see it have their results as exactly as ever. What is rounded to
    f16 is a probability (relative to the row's largest) times its page's share of R times 2^7, f16 rounds by at most 2^-25 there, and R
    is at most 16 times the largest magnitude that the row sees: keys * 2^-28 * that. (3000 tokens: keys are split over CTAs.)"""
    g = _gen(6)
    heads, blocks = 2, -(-ctx // page)
    cache = oracle.make_cache(g, blocks, heads, page, D)
    tables = oracle.tables_for(g, [ctx], page, blocks)
    first_pos = ctx - new
    at = (ctx - 1) // page                                 # a page that the last queries see
    early = max(0, first_pos - window // 2) // page        # with a window: one that only the first queries see
    cache[2][int(tables[0, at]), 0, 1] = torch.tensor(big).bfloat16().float()
    if window:
        cache[2][int(tables[0, early]), 1, 1] = torch.tensor(big).bfloat16().float()
    q = torch.randn(new, G * heads, D, generator=g).bfloat16()
    scale = D ** -0.5
    out, _ = _attend(q, cache, tables, [new], [ctx], scale, window, max_ctx=ctx)
    (o, mean, _, size), = oracle.attention(q, cache, tables, [new], [ctx], scale, window)
    m = cache[2][tables[0].long()][:, :, 1].double()       # [pages, heads]
    calm = [0, 0]
    for i in range(new):
        pos = first_pos + i
        lo = max(0, pos - window + 1) // page if window else 0
        for h in range(heads):
            seen = float(m[lo:pos // page + 1, h].max())
            calm[h] += seen < big / 2
            part = slice(h * G, h * G + G)
            oracle.assert_output(out[i:i + 1, part], o[i:i + 1, part], mean[i:i + 1, part], size, ctx * 2.0 ** -28 * seen)
    assert min(calm) > 0


# ------------------------------------------------------------------------------------------------ slots that sequences share
@pytest.mark.parametrize("new,ctx", [([1] * 200, [90] * 200), ([5] * 60, [90] * 60), ([600, 600], [700, 640])])
def test_weights_of_sequences_in_one_slot_add_up(new, ctx):
    g = _gen(7)
    heads, G, D = 2, 4, 64
    blocks = sum(-(-t // 16) for t in ctx)
    cache = oracle.make_cache(g, blocks, heads, 16, D)
    tables = oracle.tables_for(g, ctx, 16, blocks)
    q = torch.randn(sum(new), G * heads, D, generator=g).bfloat16()
    slots = _i32([1 + i % 2 for i in range(len(ctx))])
    before = torch.rand(3, heads, max(ctx), generator=g)
    _, w = _attend(q, cache, tables, new, ctx, 0.125, weights=before, slots=slots, max_ctx=max(ctx))
    want, size = before.double(), 0.0
    for b, (_, _, add, s) in enumerate(oracle.attention(q, cache, tables, new, ctx, 0.125)):
        want[int(slots[b]), :, :ctx[b]] += add
        size = max(size, s)
    oracle.assert_weights(w, want, before, size, sum(new))


# ------------------------------------------------------------------------------------------------ more new tokens than tokens
@pytest.mark.parametrize("page", [16, 32, 64])
def test_store_of_more_new_tokens_than_tokens(page):
    g = _gen(8)
    cache = oracle.make_cache(g, 12, 2, page, 64)
    new, ctx = [5, 7, 90, 65], [3, 0, 70, 64]
    tables = torch.randperm(12, generator=g).int().view(4, 3)
    lens = _i32([min(t, 3 * page) for t in ctx])
    x = torch.randn(sum(new), 4, 64, generator=g).bfloat16()
    dev, xd = _dev(*cache), x.to(DEV)
    ops.store_kv_i8(xd[:, :2], xd[:, 2:], *dev, *_dev(tables, _cu(new), lens), 90)
    _check()
    ops.store_kv_i8(x[:, :2], x[:, 2:], *cache, tables, _cu(new), lens, 90)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, cache))


# ------------------------------------------------------------------------------------------------ codes next to a tie
def _near_ties(M, per_page):
    """Numbers x = X / 2^k whose 127 x / M is a tie or next to one, and their codes, in whole numbers: twice the quotient is 254 X over
    M 2^k, and how far it is from an odd number j is |254 X - j M 2^k| / (M 2^k)."""
    found = []
    for k in range(-1, 10):
        for X in range(128, 256):
            num, den = (254 * X, M << k) if k >= 0 else (508 * X, M)
            if num > 254 * den:
                continue
            j = num // den | 1
            j = j if abs(num - j * den) <= abs(num - (j - 2) * den) else j - 2
            off, near = num - j * den, (j - 1) // 2
            code = near + (near & 1) if off == 0 else near + (off > 0)
            found.append((abs(off) / den, X / 2.0 ** k, code))
    found.sort()
    return found[:per_page]


def test_codes_of_numbers_next_to_a_tie():
    """The nearest to ties, of all significands of 8 bits: 129 / 32768 of 1 is 16383 / 32768, 2^-15 below one half."""
    assert min(abs(129 / 32768 - x / 128) for _, x, _ in _near_ties(128, 500)) == 0
    x, want = torch.zeros(128, 16, 64), torch.zeros(128, 16, 64)
    for i in range(128):
        page = _near_ties(128 + i, 510)
        v, c = torch.tensor([p[1] for p in page]), torch.tensor([float(p[2]) for p in page])
        x[i].view(-1)[:1021] = torch.cat([torch.tensor([128.0 + i]), v, -v])
        want[i].view(-1)[:1021] = torch.cat([torch.tensor([127.0]), c, -c])
    x = x.flatten(0, 1)[:, None] * 2.0 ** -7
    assert torch.equal(x.bfloat16().float(), x)
    cache = [torch.zeros(128, 1, 16, 64, dtype=torch.int8), torch.zeros(128, 1, 16, 64, dtype=torch.int8), torch.zeros(128, 1, 2)]
    args = (torch.arange(128).int()[None], _cu([2048]), _i32([2048]))
    dev = _dev(*cache)
    xd = x.bfloat16().to(DEV)
    ops.store_kv_i8(xd, -xd, *dev, *_dev(*args), 2048)
    _check()
    assert torch.equal(dev[0][:, 0].cpu().float(), want) and torch.equal(dev[1][:, 0].cpu().float(), -want)
    ops.store_kv_i8(x.bfloat16(), -x.bfloat16(), *cache, *args, 2048)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, cache))


# ------------------------------------------------------------------------------------------------ prompts in a launch chain
@pytest.mark.parametrize("ctx,new", [([300, 170], [90, 170]), ([4000, 2500], [30, 3])])
def test_prompts_and_their_weights_in_a_launch_chain(ctx, new):
    """Written, attended to, thinned out and attended to again without a wait in between; the second with keys split over CTAs."""
    from parallax_b200.ops import cuda as cu

    g = _gen(9)
    width = -(-max(ctx) // 16)
    cache = _dev(*oracle.make_cache(g, 2 * width + 20, 2, 16, 128))
    tab, new_tab = _dev(torch.arange(2 * width).int().view(2, width), (torch.arange(20) + 2 * width).int().view(2, 10))
    x = torch.randn(sum(new), 4, 128, generator=g).bfloat16().to(DEV)
    q = torch.randn(sum(new), 8, 128, generator=g).bfloat16().to(DEV)
    ends, lens, single = _dev(_cu(new), _i32(ctx), _i32([0, 1, 2]))

    def go(cache, weights):
        ops.store_kv_i8(x[:, :2], x[:, 2:], *cache, tab, ends, lens, max(new))
        out = ops.attn_prefill_i8(q, *cache, tab, ends, lens, max(new), 0.1, weights=weights)
        _, n = ops.evict_kv_i8(*cache, weights, tab, lens, new_tab, 150, 10)
        again = ops.attn_prefill_i8(q[:2], *cache, new_tab, single, n, 1, 0.1, weights=weights)
        return out, again, weights, *cache

    want = go([c.clone() for c in cache], torch.zeros(2, 2, max(ctx), device=DEV))
    _check()
    for _ in range(10):
        mine, w = [c.clone() for c in cache], torch.zeros(2, 2, max(ctx), device=DEV)
        with cu.launch_chain():
            got = go(mine, w)
        _check()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ pages of zeros
def test_codes_of_a_page_whose_magnitude_stays_are_left_as_they_are():
    """Of a magnitude of zero too: by the write and by the eviction, as the CPU forms have it."""
    g = _gen(10)
    cache = oracle.make_cache(g, 8, 2, 32, 128)
    cache[2][0] = cache[2][1, 0] = 0.0
    dev = _dev(*cache)
    x, ends, lens = torch.zeros(1, 2, 128).bfloat16(), _i32([0, 1]), _i32([40])
    tab, new_tab, weights = _i32([[1, 0]]), _i32([[2, 3]]), torch.rand(1, 2, 40, generator=g)
    d = _dev(x, tab, ends, lens, weights, new_tab)
    for c, a in ((dev, d), (cache, [x, tab, ends, lens, weights, new_tab])):
        ops.store_kv_i8(a[0], a[0], *c, *a[1:4], 1)
        ops.evict_kv_i8(*c, a[4], a[1], a[3], a[5], 35, 3)
    _check()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, cache))


# ------------------------------------------------------------------------------------------------ numbers of any size
@pytest.mark.parametrize("queries,keys", [(118, 0), (-118, 0), (120, -120), (-100, 100), (60, 40)])
@pytest.mark.parametrize("new,ctx", [([1, 1], [300, 65]), ([70, 9], [300, 65]), ([20], [3000])])
def test_weights_of_queries_and_keys_of_any_size(queries, keys, new, ctx):
    """Scores of ordinary size from numbers that are not."""
    g = _gen(11)
    blocks = sum(-(-t // 16) for t in ctx)
    cache = oracle.make_cache(g, blocks, 2, 16, 128)
    cache[2][..., 0] *= 2.0 ** keys
    tables = oracle.tables_for(g, ctx, 16, blocks)
    q = (torch.randn(sum(new), 6, 128, generator=g) * 2.0 ** queries).bfloat16()
    weights, scale = torch.rand(len(ctx), 2, max(ctx), generator=g), 0.125 * 2.0 ** -(queries + keys)
    out, w = _attend(q, cache, tables, new, ctx, scale, weights=weights, max_ctx=max(ctx))
    row = 0
    for b, (o, mean, add, size) in enumerate(oracle.attention(q, cache, tables, new, ctx, scale)):
        oracle.assert_output(out[row:row + new[b]], o, mean, size)
        want = weights[b].double()
        want[:, :ctx[b]] += add
        oracle.assert_weights(w[b], want, weights[b], size, new[b])
        row += new[b]
