"""Performance cases of the 8-bit paged key/value cache and of attention for drafted tokens.

Four operators: quantising keys and values as they are written to a paged cache and reading them back, attention of
one new token per sequence over such a cache, attention of a tree (or a chunk) of drafted tokens per sequence over a
paged cache, and committing the accepted tokens of a draft. `run` computes them in elementary torch operations, or with
`own` set through `smelt_b200.paged`.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
TOP = {"i8": 127.0, "e4m3": 448.0}  # the code of an entry's largest element


# ------------------------------------------------------------------------------------- the cases
def _store(name, seqs, low, high, q_heads, kv_heads, dim, io, cache, page, rot, style="halves", layout="hnd", start=0, pad=0):
    """`seqs` sequences of `low` to `high` new tokens, which follow `start` earlier ones each, are written and read back.
    q_heads = 0: keys and values only. `pad` further rows of the batch carry no token."""
    return {"name": name, "op": "store", "seqs": seqs, "low": low, "high": high, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "io": io, "cache": cache, "page": page, "rot": rot, "style": style, "layout": layout, "start": start, "pad": pad}


def _read(name, seqs, low, high, kv_heads, dim, io, cache, page, layout="hnd"):
    """All the tokens of `seqs` sequences are read from the cache."""
    return {"name": name, "op": "read", "seqs": seqs, "low": low, "high": high, "kv_heads": kv_heads, "dim": dim, "io": io,
            "cache": cache, "page": page, "layout": layout}


def _attend(name, seqs, low, high, q_heads, kv_heads, dim, io, cache, page, layout="hnd", window=0, empty=0):
    """`seqs` sequences of `low` to `high` cached tokens, and `empty` more without any."""
    return {"name": name, "op": "attend", "seqs": seqs, "low": low, "high": high, "empty": empty, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "io": io, "cache": cache, "page": page, "layout": layout, "window": window}


def _tree(name, seqs, low, high, nodes_low, nodes_high, q_heads, kv_heads, dim, io, cache, page, layout="hnd", chain=False, empty=0):
    """`seqs` sequences of `low` to `high` cached tokens, each followed by `nodes_low` to `nodes_high` drafted ones: of a random
    tree, or with `chain` one after the other. `empty` more sequences have no drafted token."""
    return {"name": name, "op": "tree", "seqs": seqs, "low": low, "high": high, "nodes_low": nodes_low, "nodes_high": nodes_high,
            "empty": empty, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "io": io, "cache": cache, "page": page, "layout": layout,
            "chain": chain}


def _commit(name, seqs, low, high, nodes, accepted, kv_heads, dim, cache, page, layout="hnd"):
    """`seqs` sequences of `low` to `high` cached tokens with `nodes` drafted ones each, of which up to `accepted` stay."""
    return {"name": name, "op": "commit", "seqs": seqs, "low": low, "high": high, "nodes": nodes, "accepted": accepted,
            "kv_heads": kv_heads, "dim": dim, "cache": cache, "page": page, "layout": layout}


def _spread(n, low, high):
    """n lengths from low to high, evenly spread over the logarithm, in a mixed order, mostly odd."""
    mixed = sorted(range(n), key=lambda i: (i * 37 % n, i))
    at = [(i + 0.5) / n for i in mixed]
    return [max(low, min(high, int((low + 1) * ((high + 1) / (low + 1)) ** x - 1) | 1)) for x in at]


def _lengths(c):
    return _spread(c["seqs"], c["low"], c["high"]) + [0] * (c.get("empty", 0) if c["op"] == "attend" else 0)


def _nodes(c):
    """Drafted tokens of every sequence of a tree, those of the empty ones last; their prefixes."""
    n, prefix = _spread(c["seqs"], c["nodes_low"], c["nodes_high"]), _spread(c["seqs"], c["low"], c["high"])
    return n[::-1] + [0] * c["empty"], prefix + [c["low"]] * c["empty"]


def listed():
    return [
        # one sequence's next token into an int8 cache, grouped heads: nothing but latency
        _store("store_1_token", 1, 1, 1, 32, 8, 128, "bf16", "i8", 16, 128, start=777),
        # chunked prompts of a busy server into an e4m3 cache, queries rotated on the way, half the head rotated in pairs
        _store("store_prompts", 24, 60, 2600, 32, 8, 128, "bf16", "e4m3", 16, 64, "pairs", "nhd", start=1000, pad=40),
        # one long document is taken out of the cache, to be kept elsewhere
        _read("read_document", 1, 100001, 100001, 8, 128, "bf16", "i8", 64),
        # one GPT-2 small sequence near its full context: latency
        _attend("attend_1_gpt2", 1, 1001, 1001, 12, 12, 64, "f32", "i8", 64),
        # a serving batch with grouped heads, lengths from a few tokens to thousands, one row empty
        _attend("attend_64_ragged", 63, 17, 9000, 32, 8, 128, "bf16", "i8", 16, "nhd", empty=1),
        # one long document: the work has to be split over the cache's length
        _attend("attend_long", 1, 131071, 131071, 64, 8, 128, "bf16", "e4m3", 64),
        # a small draft behind one GPT-2 small sequence: latency
        _tree("tree_1_gpt2", 1, 501, 501, 8, 8, 12, 12, 64, "f32", "f16", 64),
        # a serving batch's drafts of a few to sixty tokens, grouped heads, one sequence without a draft
        _tree("tree_32", 31, 100, 8000, 5, 60, 32, 8, 128, "bf16", "bf16", 16, "nhd", empty=1),
        # wide drafts behind long documents in an int8 cache: the work has to be split over the cache's length
        _tree("tree_long_i8", 3, 20000, 40000, 64, 64, 64, 8, 128, "bf16", "i8", 64),
        # chunks of two long prompts over what is cached of them
        _tree("chunk_2", 2, 4000, 6000, 1100, 2047, 32, 8, 128, "bf16", "bf16", 32, chain=True),
        # the accepted tokens of one small draft: latency
        _commit("commit_1_gpt2", 1, 501, 501, 8, 4, 12, 64, "f16", 64),
        # of a large batch
        _commit("commit_256", 256, 17, 900, 63, 14, 8, 128, "bf16", 16, "nhd"),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "tree", "tree", "tree", "commit"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8, 12, 16, 25])
    group = rng.choice([1, 1, 2, 4, 5, 7, 8, 16])
    eight = rng.choice(["i8", "e4m3"])
    page = rng.choice([1, 8, 16, 24, 32, 64, 128])
    layout = rng.choice(["hnd", "nhd"])
    if op == "store":
        io = rng.choice(["f32", "f16", "bf16"])
        n = _log(rng, 1, 256)
        most = min(4096, 20_000_000 // (n * dim * kv * (2 + group)))
        high = rng.choice([1, _log(rng, 1, max(1, most)), _log(rng, 1, max(1, most))])
        return _store("", n, _log(rng, 1, high), high, group * kv * rng.randint(0, 1), kv, dim, io, eight, page, rng.choice([0, dim, dim // 2]),
                      rng.choice(["halves", "pairs"]), layout, rng.choice([0, _log(rng, 1, 100_000) if n < 8 else _log(rng, 1, 999)]),
                      rng.randint(0, 9))
    if op == "read":
        n = _log(rng, 1, 256)
        high = _log(rng, 1, max(1, min(100_000, 80_000_000 // (n * dim * kv))))
        cache = rng.choice([eight, eight, "f32", "f16", "bf16"])
        return _read("", n, _log(rng, 1, high), high, kv, dim, rng.choice(["f32", "f16", "bf16"]) if SIZE[cache] == 1 else rng.choice([cache, "f32"]),
                     cache, page, layout)
    if op == "attend":
        n = _log(rng, 1, 256)
        high = _log(rng, 1, max(1, min(120_000, 130_000_000 // (n * dim * kv * max(1, group // 4)))))
        return _attend("", n, _log(rng, 1, high), high, group * kv, kv, dim, rng.choice(["f32", "f16", "bf16"]), eight, page, layout,
                       rng.choice([0, 0, _log(rng, 1, max(2, high))]), rng.choice([0, 0, rng.randint(1, 3)]))
    if op == "tree":
        cache = rng.choice([eight, "f32", "f16", "bf16", "bf16"])
        io = rng.choice(["f32", "f16", "bf16"]) if SIZE[cache] == 1 else rng.choice([cache, cache, "f32"])
        n = _log(rng, 1, 128)
        chain = rng.random() < 0.3
        nodes = _log(rng, 1, max(1, min(1000 if chain else 200, 30_000_000 // (n * kv * group * dim))))
        # scores of the plain form, and cached elements
        high = _log(rng, 1, max(1, min(60_000, 250_000_000 // (n * nodes * kv * group), 100_000_000 // (n * dim * kv))))
        return _tree("", n, rng.choice([0, _log(rng, 1, high)]), high, _log(rng, 1, nodes), nodes, group * kv, kv, dim, io, cache, page, layout,
                     chain, rng.choice([0, 0, rng.randint(1, 3)]))
    nodes = _log(rng, 1, 200)
    n = _log(rng, 1, 256)
    high = _log(rng, 1, max(1, min(4000, 40_000_000 // (n * dim * kv))))
    return _commit("", n, _log(rng, 1, high), high, nodes, rng.randint(1, nodes), kv, dim, rng.choice([eight, "f32", "f16", "bf16"]), page, layout)


def work(case):
    c = case
    b, kv, dim = SIZE.get(c.get("io"), 0), c["kv_heads"], c["dim"]
    entry = 2 * kv * (dim * SIZE[c["cache"]] + (4 if SIZE[c["cache"]] == 1 else 0))  # a token's keys and values in the cache
    if c["op"] == "store":
        n = sum(_lengths(c))
        q = n * c["q_heads"] * dim * (1 if c["rot"] else 0)
        back = SIZE[_back(c)]
        return {"bytes": n * (2 * kv * dim * (b + back) + 2 * entry + 8) + q * 2 * b,
                "flops": n * kv * dim * 10 + 3 * n * (kv + c["q_heads"]) * c["rot"]}
    if c["op"] == "read":
        n = sum(_lengths(c))
        return {"bytes": n * (entry + 2 * kv * dim * b + 8), "flops": 2 * n * kv * dim}
    if c["op"] == "attend":
        lens = _lengths(c)
        keys = sum(min(n, c["window"]) if c["window"] else n for n in lens)
        return {"bytes": keys * entry + 2 * len(lens) * c["q_heads"] * dim * b, "flops": 4 * keys * c["q_heads"] * dim}
    if c["op"] == "tree":
        nodes, prefix = _nodes(c)
        words = 0 if c["chain"] else (max(nodes) + 31) // 32
        # pairs of a token and a key that it sees; of a tree's own, a token sees itself at least
        pairs = sum(n * p + (n * (n + 1) // 2 if c["chain"] else n) for n, p in zip(nodes, prefix))
        return {"bytes": sum(n + p for n, p in zip(nodes, prefix) if n) * entry + sum(nodes) * (2 * c["q_heads"] * dim * b + 4 * words),
                "flops": 4 * pairs * c["q_heads"] * dim}
    moved = sum(_accepted(c, i) - _stay(c, i) for i in range(c["seqs"]))
    read = sum(_accepted(c, i) for i in range(c["seqs"])) * 2 * kv * dim * 2 if SIZE[c["cache"]] == 1 else 0
    return {"bytes": moved * 2 * entry + read + c["seqs"] * (8 + 4 * c["accepted"]), "flops": 0}


# ------------------------------------------------------------------------------------- the inputs
def _randn(g, *shape, kind="f32", scale=1.0):
    x = torch.empty(shape, dtype=TYPES[kind], device="cuda")
    return x.normal_(0.0, scale, generator=g)


def _quantise(x, kind):
    """Codes and scales of entries x [..., dim]: one scale per entry, which takes its largest element to the largest code."""
    top = x.abs().amax(-1)
    most = torch.full_like(top, TOP[kind])  # quotients of tensors are rounded once; those of a number and a tensor go by a reciprocal
    code = x * torch.where(top > 0, most / top, 0.0)[..., None]
    return (code.round() if kind == "i8" else code).to(TYPES[kind]), top / most


def _pool(g, c, pages):
    """Keys or values of every page as [page, head, token, dim], and their scales; in "nhd" a page holds its tokens' heads side by side."""
    nhd = c["layout"] == "nhd"
    shape = (pages, c["page"], c["kv_heads"], c["dim"]) if nhd else (pages, c["kv_heads"], c["page"], c["dim"])
    if SIZE[c["cache"]] > 1:
        codes, scales = _randn(g, *shape, kind=c["cache"]), None
    else:
        # entries of different sizes
        sizes = torch.exp(0.5 * _randn(g, *shape[:3], 1))
        codes, scales = torch.empty(shape, dtype=TYPES[c["cache"]], device="cuda"), torch.empty(shape[:3], device="cuda")
        step = max(1, 100_000_000 // max(1, codes[0].numel()))
        for at in range(0, pages, step):
            part = sizes[at : at + step]
            codes[at : at + step], scales[at : at + step] = _quantise(_randn(g, *part.shape[:3], c["dim"]) * part, c["cache"])
    if nhd:
        codes, scales = codes.transpose(1, 2), None if scales is None else scales.transpose(1, 2)
    return codes, scales


def _table(g, lens, page):
    """Pages of every sequence, drawn without order from the pool; -1 where a sequence has none. The pool's last page is nobody's."""
    need = [(n + page - 1) // page for n in lens]
    width, total = max(1, max(need)), sum(need)
    order = torch.randperm(total + 1, generator=g, device="cuda").to(torch.int32)
    order = torch.where(order == total, order[-1], order)[:total] if total else order[:0]
    first = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    column = torch.arange(width, device="cuda")
    there = column[None] < torch.tensor(need, device="cuda")[:, None]
    at = (first[:, None] + column[None]).clamp(max=max(0, total - 1))
    if not total:
        return torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"), 1
    return torch.where(there, order[at], -1).to(torch.int32).contiguous(), total + 1


def _tokens(lens, pad=0, start=0):
    """Row and position of every token of ragged sequences side by side; padding has position -1."""
    count = torch.tensor(lens + [pad], device="cuda")
    first = torch.cumsum(count, 0) - count
    row = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=sum(lens) + pad)
    real = row < len(lens)
    pos = torch.arange(sum(lens) + pad, device="cuda") - first[row] + start
    return torch.where(real, row, 0).to(torch.int32), torch.where(real, pos, -1).to(torch.int32)


def _parents(g, nodes):
    """A random tree per sequence, [sequences, nodes]: a token follows the sequence (-1) or an earlier drafted token, more often a late one."""
    i = torch.arange(max(1, max(nodes)), device="cuda")
    back = (torch.rand(len(nodes), len(i), generator=g, device="cuda") ** 2 * (i + 1)).floor().long()
    return (i - 1 - back).clamp(min=-1)


def _ancestors(parent):
    """[sequences, nodes, nodes]: whether token j lies on the way from the sequence to token i, or is i."""
    s, n = parent.shape
    seen = torch.eye(n, dtype=torch.bool, device=parent.device).expand(s, n, n).clone()
    at = parent
    for _ in range(n):
        if not bool((at >= 0).any()):
            break
        seen |= torch.nn.functional.one_hot(at.clamp(min=0), n).bool() & (at >= 0)[..., None]
        at = torch.where(at >= 0, parent.gather(1, at.clamp(min=0)), -1)
    return seen


def _words(seen):
    """Truth values [..., n] as int32 words of 32 bits, the lowest first."""
    n = seen.shape[-1]
    words = torch.nn.functional.pad(seen, (0, -n % 32)).unflatten(-1, (-1, 32)).long()
    v = (words << torch.arange(32, device=seen.device)).sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)


def _accepted(c, i):
    """How many of a sequence's drafted tokens stay."""
    return 1 + (i * 7 + 2) % c["accepted"]


def _stay(c, i):
    """How many of those are where they belong already; the others lie behind all the places that are filled."""
    n = _accepted(c, i)
    return max(min(n, i % 3), 2 * n - c["nodes"])


def _back(c):
    """The type in which what was stored is read back: a 16-bit one for rotated keys, whose rounding to 8 bits turns on the last bit of a sine."""
    return c["io"] if c["io"] != "f32" or not c["rot"] else "bf16"


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "tree":
        nodes, prefix = _nodes(c)
        total = [n + p for n, p in zip(nodes, prefix)]
    elif c["op"] == "commit":
        prefix = _lengths(c)
        total = [p + c["nodes"] for p in prefix]
    else:
        total = [n + c.get("start", 0) for n in _lengths(c)]
    s["table"], pages = _table(g, total, c["page"])
    s["k_pool"], s["k_scale"] = _pool(g, c, pages)
    s["v_pool"], s["v_scale"] = _pool(g, c, pages)
    if c["op"] in ("store", "read"):
        s["seq"], s["pos"] = _tokens(_lengths(c), c.get("pad", 0), c.get("start", 0))
    if c["op"] == "store":
        # a projection's output: queries, keys and values of a token side by side
        qkv = _randn(g, len(s["pos"]), c["q_heads"] + 2 * c["kv_heads"], c["dim"], kind=c["io"])
        s["q"] = qkv[:, : c["q_heads"]] if c["q_heads"] and c["rot"] else None
        s["k"], s["v"] = qkv[:, c["q_heads"] : c["q_heads"] + c["kv_heads"]], qkv[:, c["q_heads"] + c["kv_heads"] :]
    elif c["op"] == "attend":
        # queries of three times the unit scale: the attention rests on a few of the keys
        s["q"] = _randn(g, len(total), c["q_heads"], c["dim"], kind=c["io"], scale=3.0)
        s["lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    elif c["op"] == "tree":
        s["q"] = _randn(g, sum(nodes), c["q_heads"], c["dim"], kind=c["io"], scale=3.0)
        s["lens"] = torch.tensor(prefix, dtype=torch.int32, device="cuda")
        s["first"] = torch.tensor([0] + nodes, device="cuda").cumsum(0).to(torch.int32)
        s["mask"] = None
        if not c["chain"]:
            row, at = _tokens(nodes)
            s["mask"] = _words(_ancestors(_parents(g, nodes)))[row.long(), at.long()].contiguous()
    elif c["op"] == "commit":
        s["lens"] = torch.tensor(prefix, dtype=torch.int32, device="cuda")
        counts = torch.tensor([_accepted(c, i) for i in range(c["seqs"])], device="cuda")
        stay = torch.tensor([_stay(c, i) for i in range(c["seqs"])], device="cuda")
        # the first `stay` are 0, 1, ...; the others are drawn from the places behind
        j = torch.arange(c["nodes"], device="cuda")
        keys = torch.rand(c["seqs"], c["nodes"], generator=g, device="cuda")
        keys = torch.where(j < counts[:, None], 2.0, keys)  # places that are filled
        keys = torch.where(j < stay[:, None], -1.0, keys)
        chosen = torch.where(keys.argsort(1).argsort(1) < counts[:, None], j, c["nodes"]).sort(1).values[:, : c["accepted"]]
        s["accept"] = torch.where(torch.arange(c["accepted"], device="cuda") < counts[:, None], chosen, -1).to(torch.int32).contiguous()
        if SIZE[c["cache"]] == 1:
            s["seq"], at = _tokens(counts.tolist())
            s["pos"] = at + s["lens"][s["seq"].long()]
    if own:
        from smelt_b200.paged import PagedKV, Rotary

        s["kv"] = PagedKV(s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
        if c["op"] == "store" and c["rot"]:
            s["rotary"] = Rotary(c["rot"], 10000.0, interleaved=c["style"] == "pairs")
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


def _taken(s, c, kind):
    """The entries of tokens (seq, pos) as the values they stand for; zeros for padding."""
    pos = s["pos"].long()
    keep, at = pos >= 0, pos.clamp(min=0)
    page = s["table"][s["seq"].long(), at // c["page"]].long().clamp(min=0)
    out = []
    for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
        x = pool.view(torch.int8)[page, :, at % c["page"]].view(pool.dtype).float() if SIZE[c["cache"]] == 1 else pool[page, :, at % c["page"]].float()
        if scale is not None:
            x = x * scale[page, :, at % c["page"]][..., None]
        out.append(torch.where(keep[:, None, None], x, 0.0).to(TYPES[kind]))
    return out


def _store_plain(s, c):
    k, v, pos = s["k"], s["v"], s["pos"]
    keep = pos >= 0
    at = pos.clamp(min=0).long()
    page = s["table"][s["seq"].long(), at // c["page"]].long()
    # a row without a token writes the spare page's first entry back
    spare = s["k_pool"].shape[0] - 1
    page, at = torch.where(keep, page, spare), torch.where(keep, at % c["page"], 0)
    for pool, scales, new in ((s["k_pool"], s["k_scale"], _turn(k, pos, c)), (s["v_pool"], s["v_scale"], v.float())):
        code, scale = _quantise(new, c["cache"])
        bits = pool.view(torch.int8)
        bits[page, :, at] = torch.where(keep[:, None, None], code.view(torch.int8), bits[page, :, at])
        scales[page, :, at] = torch.where(keep[:, None], scale, scales[page, :, at])
    out = _taken(s, c, _back(c))
    if s["q"] is not None:
        out.append(_turn(s["q"], pos, c).to(s["q"].dtype))
    return out


def _gathered(s, c, width):
    """Keys and values of every row's table as fp32 [row, key, kv head, dim]."""
    out = []
    for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
        ids = s["table"].clamp(min=0).long()
        x = (pool.view(torch.int8)[ids].view(pool.dtype) if SIZE[c["cache"]] == 1 else pool[ids]).float()
        if scale is not None:
            x = x * scale[ids][..., None]
        out.append(x.transpose(2, 3).reshape(len(ids), width, c["kv_heads"], c["dim"]))
    return out


def _weighted(q, k, v, seen):
    """softmax(q k^T) v of q [row, token, head, dim], k and v [row, key, kv head, dim], seen [row, token, key]; 0 where nothing is seen."""
    n, m, heads, dim = q.shape
    kv = k.shape[2]
    qs = q.float().reshape(n, m, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, dim) / math.sqrt(dim)
    score = torch.matmul(qs, k.permute(0, 2, 3, 1)).reshape(n, kv, heads // kv, m, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3.0e38)
    e = score.sub_(top).exp_()
    total = e.sum(-1).clamp(min=1e-30)[..., None]
    o = torch.matmul(e.flatten(2, 3), v.transpose(1, 2)).reshape(n, kv, heads // kv, m, dim) / total
    return o.permute(0, 3, 1, 2, 4).reshape(n, m, heads, dim)


def _attend_plain(s, c):
    lens = s["lens"].long()
    width = s["table"].shape[1] * c["page"]
    k, v = _gathered(s, c, width)
    j = torch.arange(width, device=k.device)
    seen = j[None] < lens[:, None]
    if c["window"]:
        seen = seen & (j[None] >= lens[:, None] - c["window"])
    return _weighted(s["q"][:, None], k, v, seen[:, None])[:, 0].to(s["q"].dtype)


def _tree_plain(s, c):
    q, lens, first = s["q"], s["lens"].long(), s["first"].long()
    width = s["table"].shape[1] * c["page"]
    k, v = _gathered(s, c, width)
    n, tokens = len(lens), q.shape[0]
    m = max(1, max(_nodes(c)[0]))
    row = torch.bucketize(torch.arange(tokens, device=q.device), first[1:], right=True)
    at = torch.arange(tokens, device=q.device) - first[row]
    padded = torch.zeros(n, m, *q.shape[1:], dtype=q.dtype, device=q.device)
    padded[row, at] = q
    j = torch.arange(width, device=q.device)
    own_at = j[None] - lens[:, None]  # which drafted token a key is
    if s["mask"] is None:
        seen = own_at[:, None] <= torch.arange(m, device=q.device)[None, :, None]
    else:
        words = torch.zeros(n, m, s["mask"].shape[1], dtype=torch.int32, device=q.device)
        words[row, at] = s["mask"]
        bits = (words[..., None] >> torch.arange(32, device=q.device, dtype=torch.int32) & 1).flatten(2).bool()
        drafted = (own_at >= 0) & (own_at < bits.shape[2])
        index = own_at.clamp(0, bits.shape[2] - 1)[:, None].expand(n, m, width)
        seen = (own_at < 0)[:, None] | (bits.gather(2, index) & drafted[:, None])
    return _weighted(padded, k, v, seen)[row, at].to(q.dtype)


def _commit_plain(s, c):
    lens, accept = s["lens"].long(), s["accept"].long()
    i = torch.arange(accept.shape[1], device=lens.device)
    keep = accept >= 0
    spare = s["k_pool"].shape[0] - 1
    src, dst = lens[:, None] + accept.clamp(min=0), lens[:, None] + i

    def place(at):
        page = s["table"].gather(1, (at // c["page"]).clamp(max=s["table"].shape[1] - 1)).long()
        return torch.where(keep, page, spare), torch.where(keep, at % c["page"], 0)

    (p0, o0), (p1, o1) = place(src), place(dst)
    for pool in (s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"]):
        if pool is not None:
            bits = pool.view(torch.int8) if pool.element_size() == 1 else pool
            bits[p1, :, o1] = bits[p0, :, o0]
    new = (lens + keep.sum(1)).to(torch.int32)
    return _committed(s, c, new)


def _committed(s, c, new):
    if s["k_scale"] is None:
        return [new, s["k_pool"], s["v_pool"]]
    return [new, *(s["kv"].read(s["table"], s["pos"], s["seq"], torch.bfloat16) if own else _taken(s, c, "bf16"))]


def run(state):
    s, c = state, state["case"]
    if own:
        kv = s["kv"]
        if c["op"] == "store":
            turned = kv.append(s["k"], s["v"], s["table"], s["pos"], seq=s["seq"], rotary=s.get("rotary"), q=s["q"])
            back = kv.read(s["table"], s["pos"], s["seq"], TYPES[_back(c)])
            return [*back] + ([] if s["q"] is None else [turned])
        if c["op"] == "read":
            return [*kv.read(s["table"], s["pos"], s["seq"], TYPES[c["io"]])]
        if c["op"] == "attend":
            return kv.attend(s["q"], s["table"], s["lens"], window=c["window"])
        if c["op"] == "tree":
            return kv.attend_tree(s["q"], s["table"], s["lens"], s["first"], s["mask"])
        return _committed(s, c, kv.commit(s["table"], s["lens"], s["accept"]))
    if c["op"] == "read":
        return _taken(s, c, c["io"])
    return {"store": _store_plain, "attend": _attend_plain, "tree": _tree_plain, "commit": _commit_plain}[c["op"]](s, c)


# ------------------------------------------------------------------------------------- in 64 bits
def _exact_entries(s, c, i, positions, which):
    """Entries [position, kv head, dim] of row i in 64 bits."""
    pool, scale = s[which + "_pool"], s[which + "_scale"]
    page = s["table"][i].long()[torch.div(positions, c["page"], rounding_mode="floor")]
    x = pool.view(torch.int8)[page, :, positions % c["page"]].view(pool.dtype) if scale is not None else pool[page, :, positions % c["page"]]
    x = x.double()
    return x if scale is None else x * scale[page, :, positions % c["page"]].double().unsqueeze(-1)


def exact(case, seed):
    """The definitions, sequence by sequence, in 64 bits."""
    c, s = case, prepare(case, seed)
    if c["op"] == "store":
        r, p = c["rot"], s["pos"].double()
        real = s["pos"] >= 0
        k, q = s["k"].double(), None if s["q"] is None else s["q"].double()
        if r:
            one, two = (slice(0, r, 2), slice(1, r, 2)) if c["style"] == "pairs" else (slice(0, r // 2), slice(r // 2, r))
            theta = torch.outer(p.clamp(min=0.0), torch.exp(torch.arange(r // 2, device="cuda").double() * (-2.0 / r * math.log(10000.0))))
            turn = torch.polar(torch.ones_like(theta), theta)[:, None]
            for x in (k,) if q is None else (k, q):
                w = torch.complex(x[..., one].clone(), x[..., two].clone()) * turn
                x[..., one], x[..., two] = w.real, w.imag
        out = []
        for x in (k, s["v"].double()):
            unit = x.abs().max(-1, keepdim=True).values / TOP[c["cache"]]
            code = torch.nan_to_num(x / unit)
            code = torch.round(code) if c["cache"] == "i8" else code.float().to(torch.float8_e4m3fn).double()
            out.append(torch.where(real[:, None, None], code * unit, 0.0))
        return out + ([] if q is None else [q])
    if c["op"] == "read":
        out = [[], []]
        for i, n in enumerate(_lengths(c)):
            for o, which in zip(out, "kv"):
                o.append(_exact_entries(s, c, i, torch.arange(n, device="cuda"), which))
        return [torch.cat(o) for o in out]
    if c["op"] == "commit":
        return None
    group = c["q_heads"] // c["kv_heads"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if c["op"] == "attend":
        spans = [(i, i, i + 1, n) for i, n in enumerate(_lengths(c))]
    else:
        first = s["first"].tolist()
        spans = [(i, first[i], first[i + 1], p + m) for i, (m, p) in enumerate(zip(*_nodes(c)))]
    for i, a, b, n in spans:
        low = max(0, n - c["window"]) if c.get("window") else 0
        if a == b or n <= low:
            continue
        k, v = (_exact_entries(s, c, i, torch.arange(low, n, device="cuda"), which) for which in "kv")
        hidden = torch.zeros(b - a, n - low, dtype=torch.bool, device="cuda")
        if c["op"] == "tree":
            drafted = torch.arange(b - a, device="cuda")
            if c["chain"]:
                hidden[:, n - (b - a) :] = drafted[None] > drafted[:, None]
            else:
                hidden[:, n - (b - a) :] = torch.bitwise_and(s["mask"][a:b].long()[:, drafted // 32], (1 << (drafted % 32))[None]) == 0
        step = max(1, 200_000_000 // (n * group))
        for h in range(c["kv_heads"]):
            for at in range(0, b - a, step):
                qs = s["q"][a + at : min(b, a + at + step), h * group : (h + 1) * group].double() * c["dim"] ** -0.5
                score = torch.einsum("tgd,nd->tgn", qs, k[:, h]).masked_fill_(hidden[at : at + step, None], -math.inf)
                o[a + at : min(b, a + at + step), h * group : (h + 1) * group] = torch.einsum("tgn,nd->tgd", torch.softmax(score, -1), v[:, h])
    return o
