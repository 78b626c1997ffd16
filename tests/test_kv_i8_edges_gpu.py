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
