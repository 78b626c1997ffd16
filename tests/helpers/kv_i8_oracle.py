"""The 8-bit cache and what reads it, restated in 64 bits from the definitions, tensor by tensor on the CPU."""

import math

import torch


def make_cache(g, blocks, heads, page, D, spread=0.4):
    """A cache in use: codes of any kind, magnitudes that are bf16 numbers."""
    codes = [(torch.randn(blocks, heads, page, D, generator=g) * 45).round().clamp(-127, 127).to(torch.int8) for _ in range(2)]
    return codes[0], codes[1], torch.exp(spread * torch.randn(blocks, heads, 2, generator=g)).bfloat16().float()


def tables_for(g, lengths, page, blocks, width=None):
    """Block tables with pages in any order, none shared; what lies behind a sequence's pages is no block."""
    order = torch.randperm(blocks, generator=g).int()
    width = width or max(1, max(-(-n // page) for n in lengths))
    tables = torch.full((len(lengths), width), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        k = -(-n // page)
        tables[b, :k] = order[at:at + k]
        at += k
    assert at <= blocks
    return tables


def values(cache, table, n):
    """Keys and values ``[n, heads, D]`` of a sequence's first n tokens."""
    page = cache[0].shape[2]
    at = torch.arange(n)
    blk = table.long()[at // page]
    return [c[blk, :, at % page].double() * cache[2][blk, :, j].double()[..., None] / 127 for j, c in enumerate(cache[:2])]


def attention(q, cache, tables, new, ctx, scale, window=0, sinks=None):
    """Per sequence (output, mean magnitude of the values, weights ``[heads, tokens]``, largest sum of |q k| in log2 units)."""
    done, row = [], 0
    for b, (n, t) in enumerate(zip(new, ctx)):
        k, v = values(cache, tables[b], t)
        heads, D = k.shape[1], k.shape[2]
        x = q[row:row + n].double().view(n, heads, -1, D)
        row += n
        s = torch.einsum("qhgd,khd->qhgk", x, k) * scale
        size = torch.einsum("qhgd,khd->qhgk", x.abs(), k.abs()).nan_to_num(0, 0, 0).max() * scale * math.log2(math.e) if n * t else torch.zeros(())
        at, key = torch.arange(t - n, t)[:, None], torch.arange(t)[None]
        seen = ((key <= at) & (key > at - window) if window else key <= at)[:, None, None]
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        z = torch.logsumexp(s, -1)
        if sinks is not None:
            z = torch.logaddexp(z, sinks.double().view(1, heads, -1).expand(n, -1, -1))
        p = torch.where(seen, torch.exp(s - z[..., None]), torch.zeros_like(s))
        none = torch.isnan(v).any(-1)                                   # [tokens, heads]
        v0 = torch.where(none[..., None], torch.zeros_like(v), v)
        o, mean = torch.einsum("qhgk,khd->qhgd", p, v0), torch.einsum("qhgk,khd->qhgd", p, v0.abs())
        o[(seen[:, 0, 0, None] & none.T[None]).any(-1)] = math.nan
        done.append((o.reshape(n, -1, D), mean.reshape(n, -1, D), p.sum((0, 2)), float(size)))
    return done


def assert_output(got, want, mean, size, steps=0.0):
    """bf16 outputs: half a step of the result; and of the mean of |v|, 2^-11 for probabilities in 16 bits and the scores' error: fp32 sums
    of D products are off by up to 2^-20 of the sum of their magnitudes (`size`, in log2 units), twice that in a quotient of two sums.
    `steps`: what small probabilities lose beside pages of far larger values. What is rounded to f16 is the probability, relative to the
    row's largest or to one up to 2^8 below it, times the page's share of R, times 2^7 (decode: 2^11); f16 rounds what is too small for its
    mantissa by at most 2^-25, so a key is off by 2^-32 R (2^-36 R). The sum of the probabilities is at least 1, and R at most twice the
    largest magnitude: keys * 2^-31 (2^-35) * max |v|."""
    got, nan = got.double(), torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    far = (got - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -19 * size + 2.0 ** -14) * mean + steps + 1e-30)
    assert not (far[~nan] > 0).any(), float(far[~nan].max())


def assert_weights(got, want, before, size, queries):
    """fp32 weights: an exponential whose exponent is off by 2^-19 of `size`, 2^-18 for the exponential, the sums and the quotient, and half
    a step of every sum into a larger number."""
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    added = want.double() - before.double()
    far = (got.double() - want.double()).abs() - ((2.0 ** -19 * size + 2.0 ** -18) * added.abs() + 2.0 ** -24 * queries * want.abs() + 1e-30)
    assert not (far[~nan] > 0).any(), float(far[~nan].max())
