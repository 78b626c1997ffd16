"""Keys and values in 8 bits: what is measured of the operators that write, read, attend to and thin out such a cache.

A cache holds pages of ``page`` tokens, ``[blocks, key heads, page, dim]`` int8 codes for the keys and as many for the values, and
``kv_max`` fp32 ``[blocks, key heads, 2]``: the largest magnitude of the page's keys and of its values, head by head. A code stands for
``code * (kv_max / 127)``. Tokens that reach a page which holds some already may raise its magnitude; the codes that are there are
rounded again then: ``round(code * old / new)``.

op "append"   new tokens of every sequence into their pages, and the sequences' keys and values out again, in bf16
op "decode"   one query per sequence
op "prompt"   the queries of the last tokens of every sequence, each with the tokens up to its own
op "evict"    of every longer sequence ``keep`` tokens per key head stay: the first ``first``, the last ``recent`` and, of the others, those
              that collected the most attention. They move into pages of their own; what stayed comes out in bf16 too

Attention with ``weights`` adds to ``weights[slot, key head, token]`` what the queries of the call gave to the token, over the query heads of
the key head: what an eviction chooses by. ``run`` adds to a copy, so that it does the same every time.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------ cases
def _append(name, seqs, prefix, new, kv, dim, page):
    return dict(name=name, op="append", seqs=seqs, prefix=prefix, new=new, kv=kv, dim=dim, page=page)


def _decode(name, seqs, prefix, heads, kv, dim, page, window=0, sinks=False, weights=False):
    return dict(name=name, op="decode", seqs=seqs, prefix=prefix, new=1, heads=heads, kv=kv, dim=dim, page=page, window=window, sinks=sinks,
                weights=weights)


def _prompt(name, seqs, prefix, new, heads, kv, dim, page, window=0, sinks=False, weights=False):
    return dict(name=name, op="prompt", seqs=seqs, prefix=prefix, new=new, heads=heads, kv=kv, dim=dim, page=page, window=window, sinks=sinks,
                weights=weights)


def _evict(name, seqs, prefix, kv, dim, page, keep, recent, first):
    return dict(name=name, op="evict", seqs=seqs, prefix=prefix, new=0, kv=kv, dim=dim, page=page, keep=keep, recent=recent, first=first)


def listed():
    return [
        # a decoding batch's new tokens, one for each sequence, into pages that hold some already
        _append("append-step", 61, 150, 1, 8, 128, 16),
        # prompts of no round length
        _append("append-prompts", 3, 0, 5021, 8, 128, 64),
        # one chat
        _decode("decode-chat", 1, 776, 32, 8, 128, 16),
        # a serving batch, with what an eviction will choose by
        _decode("decode-batch-weights", 61, 2047, 32, 8, 128, 16, weights=True),
        # many long sequences, more query heads for each key head
        _decode("decode-long", 128, 12000, 40, 8, 128, 64),
        # narrow heads, a sliding window and sinks
        _decode("decode-window", 203, 3000, 64, 8, 64, 16, window=128, sinks=True),
        # a few new tokens behind a long prefix, as a follow-up question brings them
        _prompt("prompt-follow-up", 1, 30011, 37, 32, 8, 128, 16),
        # whole prompts of no round length
        _prompt("prompt-whole", 2, 0, 8111, 32, 8, 128, 64),
        # a slice of a long prompt, with what an eviction will choose by
        _prompt("prompt-slice-weights", 1, 14000, 2048, 40, 8, 128, 16, weights=True),
        # narrow heads, a sliding window and sinks
        _prompt("prompt-window", 5, 1000, 3001, 64, 8, 64, 16, window=128, sinks=True),
        # one long sequence down to an eighth
        _evict("evict-one", 1, 32767, 8, 128, 64, 4096, 1024, 4),
        # a batch of sequences that have run into their budget
        _evict("evict-batch", 40, 9000, 8, 128, 16, 2048, 500, 4),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "evict"])
    kv, dim, page = rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64])
    if op == "append":
        new = _log(rng, 1, 8000)
        seqs = max(1, min(_log(rng, 1, 200), 16000 // new))
        c = _append("", seqs, _log(rng, 1, 1000) - 1, new, kv, dim, page)
    elif op == "evict":
        prefix = _log(rng, 100, 40000)
        keep = max(24, int(prefix * rng.uniform(0.1, 0.7)))
        recent = rng.randrange(1, keep // 2)
        c = _evict("", max(1, min(_log(rng, 1, 64), 360000 // prefix)), prefix, kv, dim, page, keep, recent, rng.randrange(0, 9))
    else:
        heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        more = dict(window=rng.choice([0, 0, 0, _log(rng, 16, 4000)]), sinks=rng.random() < 0.3, weights=rng.random() < 0.3)
        if op == "decode":
            prefix = _log(rng, 1, 60000)
            c = _decode("", max(1, min(_log(rng, 1, 256), 1200000 // (prefix + 64))), prefix, heads, kv, dim, page, **more)
        else:
            new, prefix = _log(rng, 2, 6000), rng.choice([0, _log(rng, 1, 30000)])
            seqs = max(1, min(_log(rng, 1, 16), int(1.2e9 / (new * (new + prefix) * heads))))
            while seqs * new * (prefix + new / 2) * heads > 1.3e9:
                prefix //= 2
                new = new if prefix else new * 3 // 4
            c = _prompt("", seqs, prefix, new, heads, kv, dim, page, **more)
    del c["name"]
    return c


def _lengths(case):
    """New tokens and all tokens of the sequences: the first as long as the case says, the others down to a quarter of it."""
    new, total = [], []
    for i in range(case["seqs"]):
        a, b = (0.6180339887 * i) % 1.0 * 0.75, (0.7548776662 * i) % 1.0 * 0.75
        n = max(min(1, case["new"]), int(case["new"] * (1 - a)))
        new.append(n)
        total.append(max(1, n + int(case["prefix"] * (1 - b))))
    return new, total


def _pairs(case):
    """(query, key) pairs that see each other, of one head; and keys that some query sees."""
    window, pairs, keys = case["window"], 0, 0
    for n, t in zip(*_lengths(case)):
        first, w = t - n, window or t
        full = max(0, t - max(first, w - 1))               # queries with a whole window in front of them
        part = n - full                                    # these see their whole past
        pairs += full * min(w, t) + part * (first + 1 + first + part) // 2
        keys += min(t, n + w - 1)
    return pairs, keys


def work(case):
    op, kv, dim, page = case["op"], case["kv"], case["dim"], case["page"]
    new, total = _lengths(case)
    token = 2 * kv * dim                                                    # values of a token, keys and values together
    if op == "append":       # new tokens in; all codes out to the caller, the new ones into the cache
        n = sum(new)
        return {"bytes": 3 * token * n + 3 * token * sum(total) + 16 * kv * sum(-(-t // page) for t in total), "flops": 3 * token * n}
    if op == "evict":
        stay = sum(min(t, case["keep"]) for t in total)
        return {"bytes": 4 * kv * sum(total) + 4 * kv * stay + 4 * kv * sum(total) + 2 * token * stay + 3 * token * stay, "flops": token * stay}
    pairs, keys = _pairs(case)
    heads = case["heads"]
    b = token * keys + 8 * kv * keys // page + 4 * heads * dim * sum(new) + (8 * kv * keys if case["weights"] else 0)
    return {"bytes": b, "flops": 4 * heads * dim * pairs}


# ------------------------------------------------------------------------------------------------ plain form
def _scaled(codes, most):
    """Codes ``[pages, heads, page, dim]`` and magnitudes ``[pages, heads]`` -> values."""
    return codes.float() * (most / 127)[:, :, None, None]


def _sequence(s, b, n):
    """Keys and values ``[heads, n, dim]`` of a sequence's first n tokens."""
    page = s["k_cache"].shape[2]
    blocks = s["tables"][b, :-(-n // page)].long()
    most = s["kv_max"][blocks]
    return [_scaled(c[blocks], most[..., j]).transpose(0, 1).flatten(1, 2)[:, :n] for j, c in enumerate((s["k_cache"], s["v_cache"]))]


def _plain_store(s, case):
    page = case["page"]
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        if n == 0:
            continue
        p0, p1, off = (t - n) // page, (t - 1) // page + 1, (t - n) % page
        blocks = s["tables"][b, p0:p1].long()
        row = s["cu"][b]
        for j, (x, cache) in enumerate(((s["k"], s["k_cache"]), (s["v"], s["v_cache"]))):
            x = x[row:row + n].float()
            grid = x.new_zeros(((p1 - p0) * page, *x.shape[1:]))
            grid[off:off + n] = x
            grid = grid.unflatten(0, (-1, page)).transpose(1, 2)                             # [pages, heads, page, dim]
            old = s["kv_max"][blocks][..., j].clone()
            if off == 0:
                old[0] = 0.0
            old[1:] = 0.0
            most = torch.maximum(old, grid.abs().amax((2, 3)))
            safe = torch.where(most > 0, most, torch.ones_like(most))
            codes = torch.round(grid * 127 / safe[:, :, None, None])
            kept = torch.round(cache[blocks[0], :, :off].float() * old[0][:, None, None] / safe[0][:, None, None])
            codes[0, :, :off] = kept
            rows = torch.arange((p1 - p0) * page, device=DEV).view(-1, 1, page, 1)
            cache[blocks] = torch.where(rows < off + n, codes.to(torch.int8), cache[blocks])
            s["kv_max"][blocks, :, j] = most


def _plain_load(s, tables, lengths):
    at = dict(s, tables=tables)
    k, v = zip(*(_sequence(at, b, n) for b, n in enumerate(lengths)))
    return [torch.cat([x.transpose(0, 1) for x in xs]).bfloat16() for xs in (k, v)]


def _plain_attention(s, case, weights):
    q, g, scale, out = s["q"], case["heads"] // case["kv"], s["scale"], torch.empty(s["q"].shape, device=DEV, dtype=torch.bfloat16)
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        row, low = s["cu"][b], max(0, t - n - case["window"] + 1) if case["window"] else 0    # keys before `low` are behind every window
        k, v = (x[:, low:] for x in _sequence(s, b, t))
        for h in range(case["kv"]):
            x = q[row:row + n, h * g:(h + 1) * g].float().transpose(0, 1)                    # [heads, queries, dim]
            x = (x.reshape(g * n, -1) @ k[h].T).view(g, n, -1) * scale
            at, key = torch.arange(t - n, t, device=DEV)[:, None], torch.arange(low, t, device=DEV)
            seen = key <= at
            if case["window"]:
                seen = seen & (key > at - case["window"])
            x = x.masked_fill(~seen, -math.inf)
            sink = s["sinks"][h * g:(h + 1) * g, None, None] if case["sinks"] else None
            most = x.amax(-1, keepdim=True)
            most = most if sink is None else torch.maximum(most, sink)
            x = torch.exp(x - most)
            total = x.sum(-1, keepdim=True)
            total = total if sink is None else total + torch.exp(sink - most)
            x = x / total
            out[row:row + n, h * g:(h + 1) * g] = (x.view(g * n, -1) @ v[h]).view(g, n, -1).transpose(0, 1).bfloat16()
            if weights is not None:
                weights[s["slots"][b], h, low:t] += x.double().sum((0, 1)).float()
    return (out,) if weights is None else (out, weights)


def _plain_evict(s, case, weights):
    keep, recent, first, page = case["keep"], case["recent"], case["first"], case["page"]
    kept = torch.full((case["seqs"], case["kv"], keep), -1, device=DEV, dtype=torch.int32)
    lengths = [min(t, keep) for t in s["total"]]
    for b, (t, n) in enumerate(zip(s["total"], lengths)):
        row = weights[s["slots"][b]]
        if t > keep:
            best = torch.sort(row[:, first:t - recent], dim=-1, descending=True, stable=True).indices[:, :keep - first - recent] + first
            ends = torch.cat([torch.arange(first, device=DEV), torch.arange(t - recent, t, device=DEV)])
            idx = torch.cat([best, ends.expand(case["kv"], -1)], 1).sort(-1).values
        else:
            idx = torch.arange(n, device=DEV).expand(case["kv"], -1)
        kept[b, :, :n] = idx.int()
        row[:, :t] = torch.cat([row.gather(1, idx), row.new_zeros(case["kv"], t - n)], 1)
        src, pages = s["tables"][b].long()[idx // page], -(-n // page)                       # [heads, n]
        head = torch.arange(case["kv"], device=DEV)[:, None]
        to = s["new_tables"][b, :pages].long()
        for j, cache in enumerate((s["k_cache"], s["v_cache"])):
            codes, most = cache[src, head, idx % page].float(), s["kv_max"][src, head, j]    # [heads, n, dim], [heads, n]
            pad = pages * page - n
            most = torch.nn.functional.pad(most, (0, pad)).unflatten(1, (pages, page))
            codes = torch.nn.functional.pad(codes, (0, 0, 0, pad)).unflatten(1, (pages, page))
            top = most.amax(-1)
            codes = torch.round(codes * most[..., None] / torch.where(top > 0, top, torch.ones_like(top))[..., None, None])
            rows = torch.arange(pages * page, device=DEV).view(-1, 1, page, 1)
            cache[to] = torch.where(rows < n, codes.transpose(0, 1).to(torch.int8), cache[to])
            s["kv_max"][to, :, j] = top.T
    return kept, torch.tensor(lengths, device=DEV, dtype=torch.int32), weights


def _plain(s, case):
    if case["op"] == "append":
        _plain_store(s, case)
        return _plain_load(s, s["tables"], s["total"])
    weights = s["weights"].clone() if case.get("weights") or case["op"] == "evict" else None
    if case["op"] == "evict":
        done = _plain_evict(s, case, weights)
        return (*done, *_plain_load(s, s["new_tables"], [min(t, case["keep"]) for t in s["total"]]))
    return _plain_attention(s, case, weights)


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.empty(shape, device=DEV, dtype=dtype).normal_(generator=g)

    op, kv, dim, page, seqs = case["op"], case["kv"], case["dim"], case["page"], case["seqs"]
    new, total = _lengths(case)
    pages = [-(-t // page) for t in total]
    more = [-(-min(t, case["keep"]) // page) for t in total] if op == "evict" else [0] * seqs
    blocks = sum(pages) + sum(more) + 3
    order = torch.randperm(blocks, device=DEV, generator=g).int()
    s = dict(case=case, new=new, total=total, cu=[sum(new[:i]) for i in range(seqs)])
    s["tables"] = torch.zeros((seqs, max(pages) + 1), device=DEV, dtype=torch.int32)
    s["new_tables"] = torch.zeros((seqs, max(max(more), 1)), device=DEV, dtype=torch.int32)
    at = 0
    for b in range(seqs):
        s["tables"][b, :pages[b]] = order[at:at + pages[b]]
        at += pages[b]
        s["new_tables"][b, :more[b]] = order[at:at + more[b]]
        at += more[b]
    # keys and values of a trained model: normal, with some channels and tokens larger; their pages' magnitudes are bf16 numbers
    s["kv_max"] = torch.exp(0.3 * normal(blocks, kv, 2) + 1.2).bfloat16().float()
    for name in ("k_cache", "v_cache"):
        s[name] = torch.empty((blocks, kv, page, dim), device=DEV, dtype=torch.int8)
        per = max(1, (1 << 28) // (kv * page * dim))
        for i in range(0, blocks, per):
            part = s[name][i:i + per]
            part.copy_((normal(*part.shape, dtype=torch.bfloat16) * 38).round_().clamp_(-127, 127))
    s["slots"] = torch.randperm(seqs + 2, device=DEV, generator=g)[:seqs].int()
    if op == "append":
        x = normal(sum(new), 2 * kv, dim) * torch.exp(0.4 * normal(1, 2 * kv, dim))
        x = (x * torch.exp(0.3 * normal(sum(new), 1, 1))).bfloat16()
        s["k"], s["v"] = x[:, :kv], x[:, kv:]
    elif op != "evict":
        heads = case["heads"]
        s["q"] = (normal(sum(new), heads + 2 * kv, dim) * 1.5).bfloat16()[:, :heads]        # among the keys and values of a projection
        s["scale"] = dim ** -0.5
        s["sinks"] = normal(heads) if case["sinks"] else None
    if op == "evict" or case.get("weights"):
        s["weights"] = torch.exp(2.0 * normal(seqs + 2, kv, max(total) + page))
    return s


def prepare(case, seed):
    """The inputs, and the integers that a serving step keeps on the device: the ends of its sequences."""
    s = _inputs(case, seed)
    ends = [0]
    for n in (s["new"] if case["op"] != "evict" else [min(t, case["keep"]) for t in s["total"]]):
        ends.append(ends[-1] + n)
    s["cu_q"] = torch.tensor(ends, device=DEV, dtype=torch.int32)
    s["ctx"] = torch.tensor(s["total"], device=DEV, dtype=torch.int32)
    s["cu_k"] = torch.nn.functional.pad(torch.cumsum(s["ctx"], 0), (1, 0)).int()
    s["rows"], s["kept_rows"], s["max_new"], s["max_ctx"] = sum(s["total"]), ends[-1], max(s["new"]), max(s["total"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if not own:
        return _plain(s, case)
    from parallax_b200 import ops

    cache = s["k_cache"], s["v_cache"], s["kv_max"]
    if case["op"] == "append":
        ops.store_kv_i8(s["k"], s["v"], *cache, s["tables"], s["cu_q"], s["ctx"], s["max_new"])
        return ops.load_kv_i8(*cache, s["tables"], s["cu_k"], s["rows"])
    if case["op"] == "evict":
        weights = s["weights"].clone()
        kept, lengths = ops.evict_kv_i8(*cache, weights, s["tables"], s["ctx"], s["new_tables"], case["keep"], case["recent"],
                                        first=case["first"], seq_slots=s["slots"])
        return (kept, lengths, weights, *ops.load_kv_i8(*cache, s["new_tables"], s["cu_q"], s["kept_rows"]))
    more = dict(window=case["window"], sinks=s["sinks"], max_ctx=s["max_ctx"])
    if case["weights"]:
        more.update(weights=s["weights"].clone(), seq_slots=s["slots"])
    if case["op"] == "decode":
        out = ops.attn_decode_i8(s["q"], *cache, s["tables"], s["ctx"], s["scale"], **more)
    else:
        out = ops.attn_prefill_i8(s["q"], *cache, s["tables"], s["cu_q"], s["ctx"], s["max_new"], s["scale"], **more)
    return (out, more["weights"]) if case["weights"] else (out,)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_codes(s, j, block, head):
    """Codes and magnitude of one page of a head, in 64 bits."""
    return (s["k_cache"], s["v_cache"])[j][block, head].double(), s["kv_max"][block, head, j].double()


def _exact_append(s, case):
    page, out = case["page"], []
    for j, x in enumerate((s["k"], s["v"])):
        rows = []
        for b, (n, t) in enumerate(zip(s["new"], s["total"])):
            blocks = s["tables"][b, :-(-t // page)].long()
            codes, most = _exact_codes(s, j, blocks, slice(None))
            vals = torch.zeros((len(blocks) * page, case["kv"], case["dim"]), device=DEV, dtype=torch.float64)
            vals[t - n:t] = x[s["cu"][b]:s["cu"][b] + n].double()
            vals = vals.view(-1, page, case["kv"], case["dim"]).permute(0, 2, 1, 3)
            begin, first = (t - n) // page, (t - n) % page
            for p in range(begin, len(blocks)):
                old = most[p] if p == begin and first else torch.zeros_like(most[p])
                top = torch.maximum(old, vals[p].abs().amax((1, 2)))
                div = torch.where(top == 0, 1.0, top)[:, None, None]
                was = torch.round(codes[p] * old[:, None, None] / div)
                now = torch.round(127 * vals[p] / div)
                is_old = torch.arange(page, device=DEV)[:, None] < (first if p == begin else 0)
                codes[p], most[p] = torch.where(is_old, was, now), top
            v = codes * most[:, :, None, None] / 127
            rows.append(v.permute(0, 2, 1, 3).reshape(-1, case["kv"], case["dim"])[:t])
        out.append(torch.cat(rows))
    return out


def _exact_attention(s, case):
    page, g, kv = case["page"], case["heads"] // case["kv"], case["kv"]
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    weights = s["weights"].double() if case["weights"] else None
    for b, (n, t) in enumerate(zip(s["new"], s["total"])):
        blocks = s["tables"][b, :-(-t // page)].long()
        for h in range(kv):
            k, v = ((c * m[:, None, None] / 127).reshape(-1, case["dim"])[:t] for c, m in (_exact_codes(s, j, blocks, h) for j in (0, 1)))
            for r in range(0, n, 512):
                m = min(512, n - r)
                end = t - n + r + m
                low = max(0, t - n + r - case["window"] + 1) if case["window"] else 0
                q = s["q"][s["cu"][b] + r:s["cu"][b] + r + m, h * g:(h + 1) * g].double()
                x = torch.einsum("qgd,kd->gqk", q, k[low:end]) * s["scale"]
                far = torch.arange(t - n + r, end, device=DEV)[:, None] - torch.arange(low, end, device=DEV)
                x = torch.where((far >= 0) & (far < (case["window"] or t + 1)), x, -math.inf)
                z = torch.logsumexp(x, -1)
                if case["sinks"]:
                    z = torch.logaddexp(z, s["sinks"][h * g:(h + 1) * g, None].double())
                p = torch.exp(x - z[..., None])
                out[s["cu"][b] + r:s["cu"][b] + r + m, h * g:(h + 1) * g] = torch.einsum("gqk,kd->qgd", p, v[low:end])
                if weights is not None:
                    weights[s["slots"][b], h, low:end] += p.sum((0, 1))
    return (out,) if weights is None else (out, weights)


def _exact_evict(s, case):
    keep, page, weights = case["keep"], case["page"], s["weights"].double()
    values = [[], []]
    for b, t in enumerate(s["total"]):
        n, slot = min(t, keep), s["slots"][b]
        blocks = s["tables"][b, :-(-t // page)].long()
        heads = [[], []]
        for h in range(case["kv"]):
            row = weights[slot, h, :t].clone()
            if t > keep:
                rank = row.clone()
                rank[:case["first"]] = math.inf
                rank[t - case["recent"]:] = math.inf
                idx = torch.argsort(-rank, stable=True)[:n].sort().values
            else:
                idx = torch.arange(t, device=DEV)
            weights[slot, h, :t] = 0
            weights[slot, h, :n] = row[idx]
            for j in (0, 1):
                codes, most = _exact_codes(s, j, blocks, h)
                codes, most = codes.flatten(0, 1)[idx], most.repeat_interleave(page)[idx]
                for p in range(0, n, page):
                    top = most[p:p + page].max()
                    scaled = codes[p:p + page] * most[p:p + page, None]
                    codes[p:p + page] = torch.round(scaled / torch.where(top == 0, 1.0, top)) * top / 127
                heads[j].append(codes)
        for j in (0, 1):
            values[j].append(torch.stack(heads[j], 1))
    return (None, None, weights, torch.cat(values[0]), torch.cat(values[1]))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "append":
        return _exact_append(s, case)
    return _exact_evict(s, case) if case["op"] == "evict" else _exact_attention(s, case)
