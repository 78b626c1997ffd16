"""Microscaled 4-bit weights and rows: what is measured of the operators that store, expand and multiply them.

A microscaled matrix ``[rows, K]`` has one 4-bit e2m1 number per value (two per byte, the first in the low half) and one e8m0 byte
(a power of two, bias 127) per 32 values of a row:  v[r, k] = e2m1(code[r, k]) * 2^(scale[r, k / 32] - 127).

op "quantise"   rows -> codes and scales -> the values they stand for
op "product"    y = x W^T of bf16 rows and a microscaled weight, with a bias, a residual or a gate in the epilogue
op "product44"  the same with microscaled rows on both sides
op "experts"    routed feed-forward with microscaled expert matrices

A gated weight has its gate and up rows in alternating groups of 64 (``ops.interleave_gate_up``). ``act`` "silu": silu(g) u,
"clip": g = min(g, limit), u = clamp(u, -limit, limit), g sigmoid(1.702 g) (u + 1).
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
LIMIT = 7.0


# ------------------------------------------------------------------------------------------------ cases
def _quantise(name, rows, k, dtype="bf16"):
    return dict(name=name, op="quantise", rows=rows, k=k, dtype=dtype)


def _product(name, rows, n, k, bias=False, residual=False, act=""):
    return dict(name=name, op="product", rows=rows, n=n, k=k, bias=bias, residual=residual, act=act)


def _product44(name, rows, n, k, bias=False, residual=False):
    return dict(name=name, op="product44", rows=rows, n=n, k=k, bias=bias, residual=residual)


def _experts(name, rows, experts, top, k, inner, act, bias):
    return dict(name=name, op="experts", rows=rows, experts=experts, top=top, k=k, inner=inner, act=act, bias=bias)


def listed():
    return [
        # the rows of a decoding batch in front of a product of two 4-bit operands
        _quantise("rows-of-a-batch", 61, 4096),
        # a projection that is quantised when the model is loaded
        _quantise("weights-at-load", 25600, 5120, "f32"),
        # one chat: the q, k, v projection of one token
        _product("one-row", 1, 6144, 4096, bias=True),
        # a small batch: gate and up projection
        _product("few-rows-gated", 13, 51200, 5120, act="silu"),
        # a decoding batch: down projection and the residual
        _product("batch", 203, 5120, 25600, residual=True),
        # a prompt: gate and up projection
        _product("prompt-gated", 8192, 24576, 4096, act="silu"),
        # both operands in 4 bits: down projection of a decoding batch
        _product44("both-batch", 48, 4096, 12288, residual=True),
        # and one projection of a long prompt, of no round length
        _product44("both-prompt", 8111, 12288, 4096),
        # one chat on a model of 32 clipped experts
        _experts("experts-one-row", 1, 32, 4, 2880, 2880, "clip", True),
        # a decoding batch that reaches most of 128 experts
        _experts("experts-batch", 64, 128, 4, 2880, 2880, "clip", True),
        # prompts through many narrow experts
        _experts("experts-prompt-narrow", 3001, 128, 8, 2048, 768, "silu", False),
        # prompts through few wide ones
        _experts("experts-prompt-wide", 4096, 32, 4, 2880, 2880, "clip", True),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "product44", "experts"])
    if op == "quantise":
        k = 32 * _log(rng, 4, 400)
        c = _quantise("", min(_log(rng, 1, 30000), 130_000_000 // k), k, rng.choice(["bf16", "f32"]))
    elif op == "product":
        act = rng.choice(["", "", "silu", "clip"])
        k = 32 * _log(rng, 16, 800)
        n = 128 * _log(rng, 4, 400) if act else _log(rng, 500, 40000)
        n = min(n, 260_000_000 // k // 128 * 128)
        rows = min(_log(rng, 1, 8192), int(8.0e11 / (n * k)))
        c = _product("", rows, n, k, bias=rng.random() < 0.4, residual=not act and rng.random() < 0.4, act=act)
    elif op == "product44":
        k = 32 * _log(rng, 16, 600)
        n = min(_log(rng, 500, 30000), 130_000_000 // k)
        c = _product44("", min(_log(rng, 1, 8192), int(4.0e11 / (n * k))), n, k, bias=rng.random() < 0.4, residual=rng.random() < 0.4)
    else:
        act = rng.choice(["silu", "clip"])
        experts = rng.choice([8, 32, 60, 128])
        k, inner = 32 * _log(rng, 32, 100), 64 * _log(rng, 8, 50)
        c = _experts("", min(_log(rng, 1, 4096), int(8.0e11 / (experts * 0.25 * k * inner))), experts, rng.choice([1, 2, 4, 8]), k, inner, act,
                     act == "clip")
    del c["name"]
    return c


def _out_width(case):
    return case["n"] // 2 if case.get("act") else case["n"]


def work(case):
    op, t = case["op"], case["rows"]
    if op == "quantise":       # the values once in and once out, and what is stored once out and once in
        n = t * case["k"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 2 * n + 2 * (n // 2 + n // 32), "flops": 2 * n}
    if op == "experts":
        k, i, e, top = case["k"], case["inner"], case["experts"], case["top"]
        used = e * (1 - (1 - top / e) ** t)      # experts that these rows reach, on average
        per = 3 * i * k * 17 / 32 + (2 * (2 * i + k) if case["bias"] else 0)
        return {"bytes": int(used * per) + 4 * t * k + 8 * t * top, "flops": 6 * t * top * i * k}
    n, k = case["n"], case["k"]
    b = n * k * 17 // 32 + (2 * t * k if op == "product" else t * k * 17 // 32) + 2 * t * _out_width(case)
    b += 2 * n * case["bias"] + 2 * t * n * case["residual"]
    return {"bytes": b, "flops": 2 * t * n * k}


# ------------------------------------------------------------------------------------------------ plain forms
def _halves(codes):
    """Codes [..., K / 2] of two numbers each -> [..., K]."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, scales, dtype=torch.float32):
    """What codes [..., K / 2] and scales [..., K / 32] stand for."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device, dtype=dtype)
    table = torch.cat([table, -table])
    v = table[_halves(codes).int()].unflatten(-1, (-1, 32))
    power = torch.exp2(scales.to(dtype) - 127.0)
    power = torch.where(scales == 255, torch.full_like(power, math.nan), power)
    return (v * power.unsqueeze(-1)).flatten(-2)


def _codes(x):
    """Rows [R, K] -> codes [R, K / 2], scales [R, K / 32]: per 32 values the smallest power of two that keeps the largest within 6,
    then the nearest e2m1 number, ties to the even code."""
    g = x.float().unflatten(-1, (-1, 32))
    most = g.abs().amax(-1)
    part, power = torch.frexp(most)                                    # most = part * 2^power, part of [1/2, 1)
    e = torch.where(part <= 0.75, power - 3, power - 2).clamp(-127, 127)
    e = torch.where(most == 0, torch.full_like(e, -127), e)
    bad = ~torch.isfinite(most)
    q = g * torch.exp2(-e.float()).unsqueeze(-1)
    a = q.abs()
    c = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte()
         + (a > 5.0).byte())
    c = torch.where(bad.unsqueeze(-1), torch.zeros_like(c), c + 8 * torch.signbit(q).byte()).flatten(-2)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), scales


def _gate(y, act):
    """[..., N] of gate and up columns in alternating groups of 64 -> [..., N / 2]."""
    g, u = y.unflatten(-1, (-1, 2, 64)).unbind(-2)
    if act == "silu":
        return (g / (1.0 + torch.exp(-g)) * u).flatten(-2)
    g, u = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
    return (g / (1.0 + torch.exp(-1.702 * g)) * (u + 1.0)).flatten(-2)


def _plain_product(a, w, s, act):
    y = a @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].to(y.dtype)
    if s["residual"] is not None:
        y = y + s["residual"].to(y.dtype)
    return _gate(y, act) if act else y


def _plain_experts(s, case):
    """Few rows: the matrices of every row's experts side by side. Many: the rows of every expert, as many for each as the one with
    the most has."""
    t, top, k, n_exp = case["rows"], case["top"], case["k"], case["experts"]
    x, ids = s["x"].float(), s["ids"].long().flatten()                                       # [T, K], [P]
    rows = torch.arange(t * top, device=x.device) // top
    if t * top <= n_exp:
        which, a = ids, x[rows].unsqueeze(1)                                                 # [P, 1, K]
    else:
        order = torch.argsort(ids, stable=True)
        first = torch.searchsorted(ids[order], torch.arange(n_exp, device=x.device))
        place = torch.empty_like(order)
        place[order] = torch.arange(t * top, device=x.device)
        place = place - first[ids]                                                           # the pair's row of its expert
        which = torch.arange(n_exp, device=x.device)
        a = torch.zeros((n_exp, s["most"], k), device=x.device)
        a[ids, place] = x[rows]
    h = a @ _values(s["c1"][which], s["s1"][which]).transpose(1, 2)
    if s["b1"] is not None:
        h = h + s["b1"][which].float().unsqueeze(1)
    h = _gate(h, case["act"]) @ _values(s["c2"][which], s["s2"][which]).transpose(1, 2)
    if s["b2"] is not None:
        h = h + s["b2"][which].float().unsqueeze(1)
    y = h[:, 0] if t * top <= n_exp else h[ids, place]
    return s["base"].float() + (y.view(t, top, k) * s["weights"].unsqueeze(-1)).sum(1)


def _plain(s, case):
    if case["op"] == "quantise":
        return _values(*_codes(s["x"])).bfloat16()
    if case["op"] == "experts":
        return _plain_experts(s, case).bfloat16()
    a = s["x"].float() if case["op"] == "product" else _values(s["xc"], s["xs"])
    return _plain_product(a, _values(s["c"], s["s"]), s, case.get("act")).bfloat16()


# ------------------------------------------------------------------------------------------------ inputs
class _Random:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, device=DEV, dtype=dtype).normal_(0.0, std, generator=self.g)

    def rows(self, t, k):
        """Hidden states: a few channels are much larger than the others."""
        x = self.normal(t, k)
        return x * torch.exp(0.6 * self.normal(1, k, dtype=torch.float32)).bfloat16()

    def weight(self, *shape):
        """Codes and scales of normal weights, up to 2^26 of them drawn at a time."""
        *front, n, k = shape
        total = math.prod(front) * n
        per = max(1, (1 << 26) // k)
        parts = [_codes(self.normal(min(per, total - r), k, std=0.03)) for r in range(0, total, per)]
        c, s = (torch.cat(p) for p in zip(*parts))
        return c.view(*front, n, k // 2), s.view(*front, n, k // 32)


def _inputs(case, seed):
    r, t, op = _Random(seed), case["rows"], case["op"]
    if op == "quantise":
        x = r.rows(t, case["k"])
        return dict(x=x.float() * 1.01 if case["dtype"] == "f32" else x)
    if op == "experts":
        e, top, k, i = case["experts"], case["top"], case["k"], case["inner"]
        s = dict(x=r.rows(t, k), base=r.normal(t, k))
        logits = r.normal(t, e, dtype=torch.float32) + r.normal(1, e, std=0.5, dtype=torch.float32)
        best, ids = torch.topk(logits, top, dim=-1)
        s["ids"], s["weights"] = ids.int().contiguous(), torch.softmax(best, -1).contiguous()
        s["most"] = int(torch.bincount(ids.flatten()).max())
        s["c1"], s["s1"] = r.weight(e, 2 * i, k)
        s["c2"], s["s2"] = r.weight(e, k, i)
        s["b1"], s["b2"] = (r.normal(e, 2 * i, std=0.3), r.normal(e, k, std=0.3)) if case["bias"] else (None, None)
        return s
    n, k = case["n"], case["k"]
    s = dict(x=r.rows(t, k)) if op == "product" else dict(zip(("xc", "xs"), _codes(r.rows(t, k))))
    s["c"], s["s"] = r.weight(n, k)
    s["bias"] = r.normal(n, std=0.3) if case["bias"] else None
    s["residual"] = r.normal(t, n) if case["residual"] else None
    return s


def prepare(case, seed):
    """The inputs; and, as a model that has been loaded keeps them, the weights as the framework lays them out."""
    s = _inputs(case, seed)
    if own:
        from parallax_b200 import ops

        if case["op"] == "product":
            s["w"] = ops.Mx4Weight.pack(s["c"], s["s"])
        elif case["op"] == "experts":
            s["w1"], s["w2"] = (ops.Mx4Weight.pack(s[c].flatten(0, 1), s[q].flatten(0, 1), experts=case["experts"])
                                for c, q in (("c1", "s1"), ("c2", "s2")))
            s["b1"], s["b2"] = (None if b is None else b.flatten() for b in (s["b1"], s["b2"]))
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if not own:
        return _plain(s, case)
    from parallax_b200 import ops

    if case["op"] == "quantise":
        return ops.expand_mx4_rows(*ops.quant_mx4_rows(s["x"]))
    if case["op"] == "product44":
        return ops.linear_mx4_rows(s["xc"], s["xs"], s["c"], s["s"], bias=s["bias"], residual=s["residual"])
    if case["op"] == "experts":
        return ops.moe_ffn_mx4(s["x"], s["ids"], s["weights"], s["w1"], s["w2"], base=s["base"], act_mode=int(case["act"] == "clip"),
                               limit=LIMIT, b1=s["b1"], b2=s["b2"])
    epi = {"": ops.EPI_NONE, "silu": ops.EPI_SILU_MUL, "clip": ops.EPI_CLIP_GLU}[case["act"]]
    return ops.linear_mx4(s["x"], s["w"], bias=s["bias"], residual=s["residual"], epi=epi, limit=LIMIT)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _wide(codes, scales):
    """Values in 64 bits from the fields of an e2m1 number: sign, two bits of exponent, one of mantissa."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    e, m = (c // 2) % 4, c % 2
    mag = torch.where(e == 0, m.double() / 2, (1 + m.double() / 2) * 2.0 ** (e.double() - 1))
    v = torch.where(c >= 8, -mag, mag)
    p = (2.0 ** (scales.double() - 127)).masked_fill(scales == 255, math.nan)
    return v * p.repeat_interleave(32, -1)


def _wide_gate(y, act):
    b = y.reshape(y.shape[0], -1, 2, 64)
    g, u = b[:, :, 0].reshape(y.shape[0], -1), b[:, :, 1].reshape(y.shape[0], -1)
    if act == "silu":
        return torch.sigmoid(g) * g * u
    g, u = torch.clamp(g, max=LIMIT), torch.clamp(u, -LIMIT, LIMIT)
    return g * torch.sigmoid(1.702 * g) * (1 + u)


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "quantise":
        marks = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=DEV, dtype=torch.float64)
        borders = (marks[1:] + marks[:-1]) / 2
        out = torch.empty(s["x"].shape, device=DEV, dtype=torch.float64)
        for r in range(0, case["rows"], 2048):
            g = s["x"][r:r + 2048].double().unflatten(-1, (-1, 32))
            most = g.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -140)
            e = torch.ceil(torch.log2(most / 6))
            e = torch.where(most > 6 * 2.0 ** e, e + 1, torch.where(most <= 3 * 2.0 ** e, e - 1, e)).clamp(-127, 127)
            q = g / 2.0 ** e
            low = torch.bucketize(q.abs(), borders, right=False)      # a number on a border stays below it
            high = torch.bucketize(q.abs(), borders, right=True)      # or goes above
            code = torch.where(low % 2 == 0, low, high)
            out[r:r + 2048] = (torch.sign(q) * marks[code] * 2.0 ** e).flatten(-2)
        return out
    if op == "experts":
        x, ids = s["x"].double(), s["ids"].long()
        y = s["base"].double()
        for e in torch.unique(ids).tolist():
            tok, slot = torch.nonzero(ids == e, as_tuple=True)
            h = x[tok] @ _wide(s["c1"][e], s["s1"][e]).T
            h = _wide_gate(h if s["b1"] is None else h + s["b1"][e].double(), case["act"])
            h = h @ _wide(s["c2"][e], s["s2"][e]).T
            h = h if s["b2"] is None else h + s["b2"][e].double()
            y.index_add_(0, tok, h * s["weights"][tok, slot].double().unsqueeze(1))
        return y
    x = s["x"].double() if op == "product" else _wide(s["xc"], s["xs"])
    y = torch.cat([x @ _wide(c, q).T for c, q in zip(s["c"].split(4096), s["s"].split(4096))], 1)
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return _wide_gate(y, case["act"]) if case.get("act") else y
