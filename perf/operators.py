"""Performance cases of the paged key/value cache and of the token log probabilities.

Four operators: appending keys and values to a paged cache (with the position rotation), attention of
one new token per sequence over that cache, log probabilities of given tokens with entropy and top
alternatives, and their gradient. `run` computes them in elementary torch operations, or with `own` set
through `smelt_b200.paged` and `smelt_b200.logprobs`.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------- the cases
def _append(name, seqs, low, high, q_heads, kv_heads, dim, io, cache, page, rot, style="halves", layout="hnd", start=0, pad=0):
    """`seqs` sequences of `low` to `high` new tokens, which follow `start` earlier ones each. q_heads = 0: keys
    and values only. `pad` further rows of the batch carry no token."""
    return {"name": name, "op": "append", "seqs": seqs, "low": low, "high": high, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "io": io, "cache": cache, "page": page, "rot": rot, "style": style, "layout": layout, "start": start, "pad": pad}


def _attend(name, seqs, low, high, q_heads, kv_heads, dim, io, cache, page, layout="hnd", window=0, empty=0):
    """`seqs` sequences of `low` to `high` cached tokens, and `empty` more without any."""
    return {"name": name, "op": "attend", "seqs": seqs, "low": low, "high": high, "empty": empty, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "io": io, "cache": cache, "page": page, "layout": layout, "window": window}


def _logprobs(name, rows, vocab, kind, top, pad=0, temperature=1.0, masked=False):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "type": kind, "top": top, "pad": pad,
            "temperature": temperature, "masked": masked}


def _grad(name, rows, vocab, kind, pad=0, temperature=1.0, entropy=True):
    return {"name": name, "op": "grad", "rows": rows, "vocab": vocab, "type": kind, "pad": pad,
            "temperature": temperature, "entropy": entropy}


def _lengths(c):
    """The sequences' lengths: from low to high, evenly spread over the logarithm, in a mixed order, mostly odd."""
    n, low, high = c["seqs"], c["low"], c["high"]
    mixed = sorted(range(n), key=lambda i: (i * 37 % n, i))
    return [max(low, min(high, int(low * (high / low) ** ((i + 0.5) / n)) | 1)) for i in mixed] + [0] * c.get("empty", 0)


def listed():
    return [
        # one sequence's next token, grouped heads: nothing but latency
        _append("append_1_token", 1, 1, 1, 32, 8, 128, "bf16", "bf16", 16, 128, start=777),
        # a decode step of the benchmark's 32 sequences on GPT-2 small's heads: fp32 in, an fp16 cache, learned positions
        _append("append_32_gpt2", 32, 1, 1, 0, 12, 64, "f32", "f16", 64, 0, start=300),
        # chunked prompts of a busy server, queries rotated on the way, half the head rotated in pairs
        _append("append_prompts", 24, 60, 2600, 32, 8, 128, "bf16", "bf16", 16, 64, "pairs", "nhd", start=1000, pad=40),
        # one GPT-2 small sequence near its full context: latency
        _attend("attend_1_gpt2", 1, 1001, 1001, 12, 12, 64, "f32", "f16", 64),
        # the benchmark's 32 sequences over an fp32 cache, ragged
        _attend("attend_32_gpt2_f32", 32, 129, 1023, 12, 12, 64, "f32", "f32", 32),
        # a serving batch with grouped heads, lengths from a few tokens to thousands, one row empty
        _attend("attend_64_ragged", 63, 17, 9000, 32, 8, 128, "bf16", "bf16", 16, "nhd", empty=1),
        # one long document: the work has to be split over the cache's length
        _attend("attend_long", 1, 131071, 131071, 64, 8, 128, "bf16", "bf16", 64),
        # the next token of one sequence with a few alternatives
        _logprobs("logprobs_1", 1, 50257, "f32", 5),
        # a batch's sampled tokens under a temperature, a masked vocabulary, twenty alternatives
        _logprobs("logprobs_256", 256, 128000, "bf16", 20, pad=64, temperature=0.7, masked=True),
        # scoring whole documents, no alternatives
        _logprobs("logprobs_score", 4093, 50257, "f32", 0),
        # the 64 positions of the trunk backward benchmark
        _grad("grad_64", 64, 50257, "f32"),
        # a training batch
        _grad("grad_batch", 4096, 50257, "bf16", pad=7, temperature=1.3),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs", "grad"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 12, 16, 25])
    group = rng.choice([1, 1, 2, 4, 5, 7, 8, 16])
    cache = rng.choice(["f32", "f16", "bf16"])
    io = rng.choice([cache, "f32"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    layout = rng.choice(["hnd", "nhd"])
    if op == "append":
        n = _log(rng, 1, 256)
        most = min(4096, 20_000_000 // (n * dim * kv * (2 + group)))
        high = rng.choice([1, _log(rng, 1, max(1, most)), _log(rng, 1, max(1, most))])
        return _append("", n, _log(rng, 1, high), high, group * kv * rng.randint(0, 1), kv, dim, io, cache, page, rng.choice([0, dim, dim // 2]),
                       rng.choice(["halves", "pairs"]), layout, rng.choice([0, _log(rng, 1, 100_000) if n < 8 else _log(rng, 1, 999)]),
                       rng.randint(0, 9))
    if op == "attend":
        n = _log(rng, 1, 256)
        most = min(120_000, 150_000_000 // (n * dim * kv * max(1, group // 4)))
        high = _log(rng, 1, max(1, most))
        return _attend("", n, _log(rng, 1, high), high, group * kv, kv, dim, io, cache, page, layout,
                       rng.choice([0, 0, _log(rng, 1, max(2, high))]), rng.choice([0, 0, rng.randint(1, 3)]))
    kind = rng.choice(["f32", "f16", "bf16"])
    vocab = rng.choice([_log(rng, 200, 200_000), 50257])
    rows = _log(rng, 1, max(1, min(5000, 150_000_000 // vocab)))
    pad = rng.choice([0, 0, rng.randint(1, 130)])
    if op == "logprobs":
        top = rng.choice([0, 1, 5, 20, 64])
        if top:
            rows = min(rows, max(1, 60_000_000 // vocab))
        return _logprobs("", rows, vocab, kind, top, pad, rng.choice([1.0, 0.6, 1.5]), rng.random() < 0.3)
    return _grad("", rows, vocab, kind, pad, rng.choice([1.0, 0.6, 1.5]), rng.random() < 0.7)


def work(case):
    c = case
    if c["op"] == "append":
        n, b = sum(_lengths(c)), SIZE[c["io"]]
        kv, q = n * c["kv_heads"] * c["dim"], n * c["q_heads"] * c["dim"] * (1 if c["rot"] else 0)
        turned = (n * c["kv_heads"] + n * c["q_heads"]) * c["rot"]
        return {"bytes": kv * 2 * (b + SIZE[c["cache"]]) + q * 2 * b + n * 8, "flops": 3 * turned}
    if c["op"] == "attend":
        lens = _lengths(c)
        keys = sum(min(n, c["window"]) if c["window"] else n for n in lens)
        b = SIZE[c["io"]]
        return {"bytes": keys * c["kv_heads"] * c["dim"] * 2 * SIZE[c["cache"]] + 2 * len(lens) * c["q_heads"] * c["dim"] * b,
                "flops": 4 * keys * c["q_heads"] * c["dim"]}
    n, b = c["rows"] * c["vocab"], SIZE[c["type"]]
    if c["op"] == "logprobs":
        return {"bytes": n * b + c["rows"] * (16 + 8 * c["top"]), "flops": 5 * n}
    return {"bytes": 2 * n * b + c["rows"] * 24, "flops": 6 * n}


# ------------------------------------------------------------------------------------- the inputs
def _randn(g, *shape, kind="f32", scale=1.0):
    x = torch.empty(shape, dtype=TYPES[kind], device="cuda")
    return x.normal_(0.0, scale, generator=g)


def _pool(g, c, pages):
    """Keys or values of every page, as [page, head, token, dim]; a page holds its tokens' heads side by side in "nhd"."""
    if c["layout"] == "hnd":
        return _randn(g, pages, c["kv_heads"], c["page"], c["dim"], kind=c["cache"])
    return _randn(g, pages, c["page"], c["kv_heads"], c["dim"], kind=c["cache"]).transpose(1, 2)


def _table(g, lens, page):
    """Pages of every sequence, drawn without order from the pool; -1 where a sequence has none. The pool's last page is nobody's."""
    need = [(n + page - 1) // page for n in lens]
    width, total = max(1, max(need)), sum(need)
    order = torch.randperm(total + 1, generator=g, device="cuda").to(torch.int32)
    order = torch.where(order == total, order[-1], order)[:total] if total else order[:0]
    own_from = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    column = torch.arange(width, device="cuda")
    there = column[None] < torch.tensor(need, device="cuda")[:, None]
    at = (own_from[:, None] + column[None]).clamp(max=max(0, total - 1))
    if not total:
        return torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"), 1
    return torch.where(there, order[at], -1).to(torch.int32).contiguous(), total + 1


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] in ("append", "attend"):
        lens = _lengths(c)
        s["table"], pages = _table(g, [n + c.get("start", 0) for n in lens], c["page"])
        s["k_pool"], s["v_pool"] = _pool(g, c, pages), _pool(g, c, pages)
        if own:
            from smelt_b200.paged import PagedKV, Rotary

            s["kv"] = PagedKV(s["k_pool"], s["v_pool"])
            if c["op"] == "append" and c["rot"]:
                s["rotary"] = Rotary(c["rot"], 10000.0, interleaved=c["style"] == "pairs")
    if c["op"] == "append":
        n, pad = sum(lens), c["pad"]
        count = torch.tensor(lens + [pad], device="cuda")
        first = torch.cumsum(count, 0) - count
        row = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=n + pad)
        real = row < len(lens)
        pos = torch.arange(n + pad, device="cuda") - first[row] + c["start"]
        s["pos"] = torch.where(real, pos, -1).to(torch.int32)
        s["seq"] = torch.where(real, row, 0).to(torch.int32)
        # a projection's output: queries, keys and values of a token side by side
        heads = c["q_heads"] + 2 * c["kv_heads"]
        qkv = _randn(g, n + pad, heads, c["dim"], kind=c["io"])
        s["q"] = qkv[:, : c["q_heads"]] if c["q_heads"] else None
        s["k"], s["v"] = qkv[:, c["q_heads"] : c["q_heads"] + c["kv_heads"]], qkv[:, c["q_heads"] + c["kv_heads"] :]
    elif c["op"] == "attend":
        # queries of three times the unit scale: the attention rests on a few of the keys
        s["q"] = _randn(g, len(lens), c["q_heads"], c["dim"], kind=c["io"], scale=3.0)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    else:
        rows, vocab = c["rows"], c["vocab"]
        x = _randn(g, rows, vocab + c["pad"], kind=c["type"], scale=2.5)[:, :vocab]
        t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        if c.get("masked"):
            hidden = torch.rand(vocab, generator=g, device="cuda") < 0.5
            x.masked_fill_(hidden[None], -math.inf)
            t = torch.where(hidden[t], (~hidden).int().argmax(), t)
        # the given token is a likely one
        x[torch.arange(rows, device="cuda"), t] = _randn(g, rows, kind=c["type"], scale=3.0) + 8.0
        s["logits"], s["targets"] = x, t.to(torch.int32)
        if c["op"] == "grad":
            s["d_lp"] = _randn(g, rows)
            s["d_entropy"] = _randn(g, rows) if c["entropy"] else None
            # what the forward pass left: the largest logit, the logarithm of the sum, the entropy
            z = (x.float() - x.float().amax(1, keepdim=True)) / c["temperature"]
            total = z.exp().sum(1)
            s["stats"] = torch.stack([x.float().amax(1), total.log(), total.log() - (z.exp() * z).sum(1) / total], 1).contiguous()
    return s


# ------------------------------------------------------------------------------------- one pass
def _turn(x, pos, c, base=10000.0):
    """x [token, head, dim] rotated by its token's position; a token without one is left as it is."""
    r = c["rot"]
    if not r:
        return x.float()
    f = base ** (-torch.arange(0, r, 2, device=x.device, dtype=torch.float64) / r)
    angle = pos.clamp(min=0).double()[:, None, None] * f
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    y = x.float().clone()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if c["style"] == "pairs" else (y[..., : r // 2], y[..., r // 2 : r])
    turned = a * cos - b * sin, b * cos + a * sin
    a.copy_(turned[0]), b.copy_(turned[1])
    return y


def _append_plain(s, c):
    k, v, pos = s["k"], s["v"], s["pos"]
    keep = pos >= 0
    at = pos.clamp(min=0).long()
    page = s["table"][s["seq"].long(), at // c["page"]].long()
    # a row without a token writes the spare page's first entry back
    spare = s["k_pool"].shape[0] - 1
    page, at = torch.where(keep, page, spare), torch.where(keep, at % c["page"], 0)
    for pool, new in ((s["k_pool"], _turn(k, pos, c)), (s["v_pool"], v.float())):
        pool[page, :, at] = torch.where(keep[:, None, None], new.to(pool.dtype), pool[page, :, at])
    out = [s["k_pool"], s["v_pool"]]
    if s["q"] is not None and c["rot"]:
        out.append(_turn(s["q"], pos, c).to(s["q"].dtype))
    return out


def _attend_plain(s, c):
    q, lens = s["q"], s["lens"].long()
    n, page, kv, dim = q.shape[0], c["page"], c["kv_heads"], c["dim"]
    width = s["table"].shape[1] * page
    k, v = (p[s["table"].clamp(min=0).long()].transpose(2, 3).reshape(n, width, kv, dim) for p in (s["k_pool"], s["v_pool"]))
    j = torch.arange(width, device=q.device)
    seen = j[None] < lens[:, None]
    if c["window"]:
        seen = seen & (j[None] >= lens[:, None] - c["window"])
    qs = q.float().reshape(n, kv, -1, dim) / math.sqrt(dim)
    score = torch.matmul(qs, k.float().permute(0, 2, 3, 1)).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3.0e38)
    e = torch.exp(score - top)
    o = torch.matmul(e, v.float().transpose(1, 2)) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(n, c["q_heads"], dim).to(q.dtype)


def _logprobs_plain(s, c):
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    z = (x - m) / c["temperature"]
    e = z.exp()
    total = e.sum(1)
    t = s["targets"].long()[:, None]
    lp = z.gather(1, t)[:, 0] - total.log()
    entropy = total.log() - (e * z.clamp(min=-1000.0)).sum(1) / total
    out = {"lp": lp, "entropy": entropy}
    if c["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : c["top"]]
        out["top_ids"] = ids.to(torch.int32)
        out["top_lp"] = z.gather(1, ids) - total.log()[:, None]
    return out


def _grad_plain(s, c):
    x = s["logits"].float()
    m, log_sum, entropy = s["stats"].unbind(1)
    lp = (x - m[:, None]) / c["temperature"] - log_sum[:, None]
    p = lp.exp()
    d = -s["d_lp"][:, None] * p
    d.scatter_add_(1, s["targets"].long()[:, None], s["d_lp"][:, None])
    if s["d_entropy"] is not None:
        d = d - s["d_entropy"][:, None] * p * (lp + entropy[:, None])
    return (d / c["temperature"]).to(s["logits"].dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        if c["op"] == "append":
            q = s["q"] if c["rot"] else None
            turned = s["kv"].append(s["k"], s["v"], s["table"], s["pos"], seq=s["seq"], rotary=s.get("rotary"), q=q)
            return [s["k_pool"], s["v_pool"]] + ([] if q is None else [turned])
        if c["op"] == "attend":
            return s["kv"].attend(s["q"], s["table"], s["lens"], window=c["window"])
        from smelt_b200.logprobs import token_logprobs, token_logprobs_grad

        if c["op"] == "logprobs":
            r = token_logprobs(s["logits"], s["targets"], top=c["top"], temperature=c["temperature"])
            out = {"lp": r.lp, "entropy": r.entropy}
            return out | {"top_ids": r.top_ids, "top_lp": r.top_lp} if c["top"] else out
        return token_logprobs_grad(s["logits"], s["targets"], s["stats"], s["d_lp"], s["d_entropy"], temperature=c["temperature"])
    return {"append": _append_plain, "attend": _attend_plain, "logprobs": _logprobs_plain, "grad": _grad_plain}[c["op"]](s, c)


# ------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions, sequence by sequence or a block of rows at a time, in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["op"] == "append":
        pools = [s["k_pool"].double(), s["v_pool"].double()]
        n = sum(_lengths(c))  # the padding comes last
        p = s["pos"][:n].double()
        r = c["rot"]
        k, q = s["k"][:n].double(), (s["q"].double() if s["q"] is not None else None)
        if r:
            first, second = (slice(0, r, 2), slice(1, r, 2)) if c["style"] == "pairs" else (slice(0, r // 2), slice(r // 2, r))
            theta = torch.outer(p, torch.exp(torch.arange(r // 2, device="cuda").double() * (-2.0 / r * math.log(10000.0))))
            turn = torch.polar(torch.ones_like(theta), theta)[:, None]
            for x in (k,) + ((q[:n],) if q is not None else ()):
                w = torch.complex(x[..., first].clone(), x[..., second].clone()) * turn
                x[..., first], x[..., second] = w.real, w.imag
        where = s["pos"][:n].long()
        flat = s["table"].long().reshape(-1)[s["seq"][:n].long() * s["table"].shape[1] + torch.div(where, c["page"], rounding_mode="floor")]
        for pool, x in zip(pools, (k, s["v"][:n].double())):
            pool.index_put_((flat[:, None], torch.arange(c["kv_heads"], device="cuda")[None], (where % c["page"])[:, None]), x)
        return pools + ([q] if q is not None and r else [])
    if c["op"] == "attend":
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = c["q_heads"] // c["kv_heads"]
        for i, n in enumerate(_lengths(c)):
            if not n:
                continue
            pages = s["table"][i, : (n + c["page"] - 1) // c["page"]].long()
            low = max(0, n - c["window"]) if c["window"] else 0
            for h in range(c["kv_heads"]):
                k, v = (x[pages, h].reshape(-1, c["dim"])[low:n].double() for x in (s["k_pool"], s["v_pool"]))
                score = s["q"][i, h * group : (h + 1) * group].double() @ k.T * c["dim"] ** -0.5
                o[i, h * group : (h + 1) * group] = torch.softmax(score, -1) @ v
        return o
    blocks = []
    step = max(1, 40_000_000 // c["vocab"])
    for at in range(0, c["rows"], step):
        x = s["logits"][at : at + step].double() / c["temperature"]
        t = s["targets"][at : at + step].long()
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        h = torch.special.entr(p).sum(1)
        if c["op"] == "logprobs":
            one = {"lp": lp[torch.arange(len(t), device="cuda"), t], "entropy": h}
            if c["top"]:
                one["top_lp"] = lp.topk(c["top"], 1).values
            blocks.append(one)
        else:
            d = -s["d_lp"][at : at + step, None].double() * p
            d[torch.arange(len(t), device="cuda"), t] += s["d_lp"][at : at + step].double()
            if s["d_entropy"] is not None:
                d -= s["d_entropy"][at : at + step, None].double() * (p * h[:, None] - torch.special.entr(p))
            blocks.append(d / c["temperature"])
    if c["op"] == "grad":
        return torch.cat(blocks)
    out = {key: torch.cat([b[key] for b in blocks]) for key in blocks[0]}
    if c["top"]:
        out["top_ids"] = None
    return out
