"""Microscaled 4-bit operators in 64 bits, element by element from their definition, with bounds on what a kernel may be off by.

Roundings are counted as half a step of their type (bf16: 2^-8 of the value). A sum of n products that are exact in fp32 and are
added in fp32 in any order, with truncation, is off by at most n * 2^-23 times the sum of their magnitudes."""

import torch

BF16 = 2.0 ** -8
MAGS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def values(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(c >= 8, -MAGS[c % 8], MAGS[c % 8])
    p = torch.pow(2.0, scales.double() - 127).masked_fill(scales == 255, float("nan"))
    return v * p.repeat_interleave(32, -1)


def quantise(x):
    """(values, exponents, whether the group is finite) by search over all powers and all eight magnitudes."""
    g = x.double().unflatten(-1, (-1, 32))
    most = g.abs().amax(-1)
    powers = torch.arange(-127, 128, dtype=torch.float64)
    e = powers[(most.unsqueeze(-1) <= 6 * 2.0 ** powers).int().argmax(-1)]       # the smallest that fits
    q = g / (2.0 ** e).unsqueeze(-1)
    d = (q.abs().unsqueeze(-1) - MAGS).abs()
    near = d == d.amin(-1, keepdim=True)
    first, last = near.int().argmax(-1), 7 - near.flip(-1).int().argmax(-1)
    code = torch.where(first % 2 == 0, first, last)                              # a tie lies between an even and an odd code
    return (torch.sign(q) * MAGS[code] * (2.0 ** e).unsqueeze(-1)).flatten(-2), e, torch.isfinite(most)


def product(x, w, bias=None):
    """(x W^T + bias, bound of a sum in fp32) of 64-bit matrices."""
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, s = y + bias.double(), s + bias.double().abs()
    return y, (x.shape[1] + 2) * 2.0 ** -23 * s


def gate(y, ey, clip, limit):
    """The gated columns of (y, bound), gate / up in groups of 64. Both activations have a slope of at most 1.1 in the gate; the
    exponential, the division and the products are off by 2^-19 of the result."""
    b, eb = y.unflatten(-1, (-1, 2, 64)), ey.unflatten(-1, (-1, 2, 64))
    (g, u), (eg, eu) = ((t[..., 0, :].flatten(-2), t[..., 1, :].flatten(-2)) for t in (b, eb))
    if clip:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
        s = g * torch.sigmoid(1.702 * g)
    else:
        s = g * torch.sigmoid(g)
    return s * u, 1.1 * eg * u.abs() + s.abs() * eu + 1.1 * eg * eu + 2.0 ** -19 * (s * u).abs()


def linear(x, w, bias=None, residual=None, act="", limit=7.0):
    y, e = product(x, w, bias)
    if act:
        y, e = gate(y, e, act == "clip", limit)
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return y, e + BF16 * (y.abs() + e)


def experts(x, ids, weights, w1, w2, base, clip, limit, b1, b2):
    """w1 [E, 2 I, K], w2 [E, K, I] in 64 bits."""
    out = base.double().clone() if base is not None else torch.zeros_like(x, dtype=torch.float64)
    err = torch.zeros_like(out)
    size = out.abs()
    for e in range(w1.shape[0]):
        tok, slot = (ids == e).nonzero(as_tuple=True)
        if not tok.numel():
            continue
        h, eh = gate(*product(x[tok].double(), w1[e], None if b1 is None else b1[e]), clip, limit)
        eh = eh + BF16 * (h.abs() + eh)                                          # the rows between the products are bf16
        y, ey = product(h, w2[e], None if b2 is None else b2[e])
        ey = ey + (1 + 2.0 ** -10) * (eh @ w2[e].abs().t())
        f = weights[tok, slot].double().unsqueeze(1)
        out.index_add_(0, tok, f * y)
        err.index_add_(0, tok, f.abs() * ey)
        size.index_add_(0, tok, (f * y).abs())
    err = err + (ids.shape[1] + 1) * 2.0 ** -23 * (size + err)
    return out, err + BF16 * (out.abs() + err)


def within(got, want, bound, what=""):
    """got is within the bound everywhere; NaN and infinities are where they are expected."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN in other places")
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), (what, "infinities differ")
    far = ((got - want).abs() - bound)[fine]
    assert not far.numel() or float(far.max()) <= 0, (what, "over the bound by", float(far.max()))
