"""Attention of drafted tokens over paged caches against 64 bits (paged_oracle.py derives the bounds), committing a draft, and a
speculative step of both with append and read."""
import math

import numpy as np
import pytest
import torch

from smelt_b200._ffi import Gpt2qError
from smelt_b200.paged import STATUS_PAGE, STATUS_POSITION, PagedKV, Rotary, tree_mask

from .paged_oracle import T, U, WEIGHT, Cache, attention64, bound_of, close, gen, randn, tables

pytestmark = pytest.mark.gpu
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "i8"), ("bf16", "i8"), ("f16", "i8"),
         ("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e4m3")]


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def bits(x):
    return x.view(torch.int8) if x.element_size() == 1 else x


def random_tree(rng, n):
    return [-1 if rng.random() < 0.1 else int(rng.integers(max(-1, i - 6), i)) for i in range(n)]


def seen_by(mask, a, b, keys, prefix):
    """[tokens, keys]: what the tokens a..b-1 of one row see of the row's positions."""
    m = b - a
    own = keys - prefix
    if mask is None:
        return own[None] <= torch.arange(m, device="cuda")[:, None]
    words = mask[a:b].long()
    inside = (own >= 0) & (own < words.shape[1] * 32)
    j = own.clamp(0, words.shape[1] * 32 - 1)
    bit = (words[:, j // 32] >> (j % 32)) & 1 == 1
    return (own < 0)[None] | (bit & inside[None])


def tree_case(seed, prefixes, nodes, heads, kv, dim, io, cache, page, layout="hnd", chain=False, gap=0, scale=3.0, words=None, mask=None, sizes=0.5,
              spoil=True, sm=None):
    """`gap` tokens before the first row and two behind the last belong to none."""
    g, rng = gen(seed), np.random.default_rng(seed)
    there = [max(0, p) + n if n else 0 for p, n in zip(prefixes, nodes)]
    pages = sum(-(-n // page) for n in there) + 1
    c = Cache(g, pages, kv, page, dim, cache, layout, sizes)
    table = tables(rng, there, page, pages)
    values = c.values
    if spoil:
        c.spoil(c.used(table, there))
    first = np.cumsum([gap] + nodes)
    total = int(first[-1]) + (2 if gap else 0)
    if mask is None and not chain:
        m, _ = tree_mask([random_tree(rng, n) for n in nodes])
        mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (total, m.shape[1]), dtype=torch.int32, device="cuda", generator=g)
        mask[gap:gap + len(m)] = m
        if words:
            mask = torch.nn.functional.pad(mask, (0, words - mask.shape[1])) if words > mask.shape[1] else mask[:, :words].contiguous()
    q = randn(g, total, heads, dim, kind=io, scale=scale)
    lse = torch.full((total, heads), 7.0, device="cuda")
    out = torch.full_like(q, 9.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    sm = dim ** -0.5 if sm is None else sm
    r = c.kv.attend_tree(q, table, i32(prefixes), i32(first), mask, scale=sm, out=out, lse=lse, status=status)
    assert r is out and int(status) == 0
    for k, (p, n) in enumerate(zip(prefixes, nodes)):
        a, b = int(first[k]), int(first[k + 1])
        if a == b:
            continue
        keys = torch.arange(there[k], device="cuda")
        seen = seen_by(mask, a, b, keys, max(0, p))
        want, wl, tol, size, rel, vmax = attention64(q[a:b], values, table[k], keys, seen, sm)
        close(out[a:b], want, bound_of(tol, size, vmax, want, io, cache, wide=True), ("out", k))
        fin = torch.isfinite(wl)
        assert torch.equal(fin, torch.isfinite(lse[a:b])) and bool((lse[a:b][~fin] == -math.inf).all())
        assert bool((out[a:b][~fin] == 0).all())
        close(lse[a:b][fin], wl[fin], (rel + (wl.abs() + 1) * 4 * U + 2.0 ** -20)[fin] + (0 if io == "f32" else 1.01 * WEIGHT[cache == "bf16"]), ("lse", k))
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    inside[gap:int(first[-1])] = True
    assert bool((out[~inside] == 9.0).all()) and bool((lse[~inside] == 7.0).all())
    return out


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (8, 2), (7, 1), (16, 1), (40, 2), (15, 5)])
def test_heads_and_types(io, cache, heads, kv):
    tree_case(1, [33, 0, 5, 200, 16], [7, 1, 0, 33, 16], heads, kv, 64, io, cache, 16, gap=3)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 144, 192, 256])
@pytest.mark.parametrize("page,chain", [(24, False), (32, True), (16, False)])
def test_head_dims(io, cache, dim, page, chain):
    tree_case(2, [70, 31, -3, 129], [9, 1, 20, 5], 6, 2, dim, io, cache, page, "nhd", chain)


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 24, 40, 200])
def test_head_dims_that_are_no_multiple_of_16(cache, dim):
    tree_case(3, [70, 3], [9, 12], 6, 2, dim, cache, cache, 16)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("page", [1, 3, 16, 64, 1000])
@pytest.mark.parametrize("chain", [False, True])
def test_pages(io, cache, page, chain):
    tree_case(4, [15, 16, 17, 255, 1, 300, 0], [1, 16, 15, 2, 64, 3, 5], 4, 4, 64, io, cache, page, chain=chain)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("prefixes,nodes", [([9001], [40]), ([3] * 700, [1] * 700), ([4097, 1, 0, 3000, 64], [64, 0, 130, 1, 17]), ([0, 0], [0, 0]),
                                            ([100], [1]), ([2000] * 3, [257, 100, 300])])
@pytest.mark.parametrize("chain", [False, True])
def test_long_and_many(io, cache, prefixes, nodes, chain):
    tree_case(5, prefixes, nodes, 8, 2, 128, io, cache, 16, chain=chain, scale=1.0)


@pytest.mark.parametrize("io,cache", TYPES)
def test_masks_of_other_widths_and_without_bits(io, cache):
    """Words past the tokens, tokens past the words, tokens that see nothing at all or only what is no tree."""
    tree_case(6, [40, 3], [30, 9], 4, 2, 64, io, cache, 16, words=3)
    tree_case(7, [40, 0], [70, 9], 4, 2, 64, io, cache, 16, words=1)
    mask = torch.zeros(50, 2, dtype=torch.int32, device="cuda")
    tree_case(8, [0, 20, 0], [10, 30, 10], 4, 2, 64, io, cache, 16, mask=mask)
    mask[::3, 0] = -(2 ** 31)   # token 31 alone
    mask[1::3, 1] = 2 ** 30     # one that no row has
    mask[2::3, 0] = 0x155       # whatever comes later
    tree_case(9, [0, 20, 0], [10, 32, 8], 4, 2, 64, io, cache, 16, mask=mask)


@pytest.mark.parametrize("io,cache", TYPES)
def test_what_is_not_seen_does_not_reach_a_token(io, cache):
    """Infinities and NaN in the keys and values of drafted tokens: those that see one give NaN, the others are as without it."""
    g, rng = gen(10), np.random.default_rng(10)
    page, prefix, n, dim = 16, 37, 80, 64
    c = Cache(g, 9, 2, page, dim, cache)
    table = tables(rng, [prefix + n], page, 9)
    parents = random_tree(rng, n)
    mask, _ = tree_mask([parents])
    q = randn(g, n, 8, dim, kind=io)
    args = (q, table, i32([prefix]), i32([0, n]), mask)
    clean = c.kv.attend_tree(*args)
    bits_of = mask.cpu().numpy().view(np.uint32)
    for which, node, what in ((0, 5, math.nan), (1, 11, math.nan), (1, 30, math.inf), (1, 70, -math.inf), (0, 75, math.inf)):
        slot = (table[0, (prefix + node) // page].item(), slice(None), (prefix + node) % page)
        if c.scales[which] is not None:
            hold = c.scales[which][slot].clone()
            c.scales[which][slot] = math.nan
        else:
            hold = c.pools[which][slot].clone()
            c.pools[which][slot[0], :, slot[2], 3] = what
        out = c.kv.attend_tree(*args)
        sees = torch.tensor([bool(bits_of[t, node // 32] >> (node % 32) & 1) for t in range(n)], device="cuda")
        assert torch.equal(out[~sees], clean[~sees])
        if which == 1 or math.isnan(what) or cache in ("i8", "e4m3"):
            assert bool(torch.isnan(out[sees]).flatten(1).all()) if which == 0 else bool(torch.isnan(out[sees]).flatten(1).any(1).all())
        if c.scales[which] is not None:
            c.scales[which][slot] = hold
        else:
            c.pools[which][slot] = hold
    assert torch.equal(c.kv.attend_tree(*args), clean)


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
def test_scales_of_very_different_sizes(cache, io):
    tree_case(11, [700, 64, 33], [40, 64, 5], 8, 2, 64, io, cache, 16, scale=1e-3, sizes=4.0)


@pytest.mark.parametrize("io,cache", TYPES)
def test_extreme_scores_and_scales(io, cache):
    for scale, sm in ((300.0, None), (1e-4, None), (3.0, -0.1), (3.0, 0.0)):
        tree_case(12, [77, 300], [9, 70], 4, 1, 64, io, cache, 16, scale=scale, sm=sm)


@pytest.mark.parametrize("io,cache", TYPES)
def test_bad_pages_and_lengths_give_nan(io, cache):
    g = gen(14)
    c = Cache(g, 6, 2, 16, 64, cache)
    table = i32([[0, 1, -1], [2, 6, 3], [4, 5, 0], [5, 7, 9]])
    q = randn(g, 40, 4, 64, kind=io)

    def run(lens, nodes):
        first = i32(np.cumsum([0] + nodes))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lse = torch.empty(40, 4, device="cuda")
        o = c.kv.attend_tree(q, table, i32(lens), first, None, lse=lse, status=status)
        nan = torch.isnan(o).flatten(1)
        rows = [nan[int(first[i]):int(first[i + 1])] for i in range(4)]
        assert all(bool(r.all()) == bool(r.any()) for r in rows if len(r))
        return [bool(r.any()) for r in rows], int(status)
    assert run([22, 6, 38, 0], [10, 10, 10, 0]) == ([False, False, False, False], 0)
    assert run([23, 7, 38, 6], [10, 10, 10, 10]) == ([True, True, False, False], STATUS_PAGE)
    assert run([22, 38, 39, 1], [10, 10, 10, 10]) == ([False, True, True, False], STATUS_PAGE | STATUS_POSITION)
    assert run([22, 2 ** 31 - 1, 39, 1], [10, 10, 10, 10]) == ([False, True, True, False], STATUS_PAGE | STATUS_POSITION)
    assert run([400, 900, 39, 1], [0, 0, 0, 10]) == ([False, False, False, False], 0)  # rows without drafted tokens are not looked at


@pytest.mark.parametrize("io,cache", [("bf16", "bf16"), ("f32", "f16"), ("bf16", "i8")])
def test_first_that_does_not_rise_stays_in_bounds(io, cache):
    """A malformed `first` may give any numbers, but nothing outside the tensors is touched."""
    g = gen(15)
    c = Cache(g, 8, 2, 16, 64, cache)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    hold = torch.full((40, 4, 64), 5.0, dtype=T[io], device="cuda")
    q, out = randn(g, 20, 4, 64, kind=io), hold[10:30]
    for first in ([-7, 12, 5], [15, 3, 900], [2 ** 31 - 1, -2 ** 31, 0], [0, 2 ** 30, 2 ** 31 - 1]):
        c.kv.attend_tree(q, table, i32([20, 30]), i32(first), None, out=out)
        assert bool((hold[:10] == 5.0).all()) and bool((hold[30:] == 5.0).all())


def test_strided_queries_outputs_table_and_offsets_past_32_bits():
    pages, page, dim = 1100, 32, 128
    stride = 1 << 22  # elements between pages: page 1025 starts past 2^32
    store = torch.empty(pages * stride, dtype=torch.bfloat16, device="cuda")
    k_pool = store.as_strided((pages, 2, page, dim), (stride, page * dim, dim, 1))
    v_pool = store.as_strided((pages, 2, page, dim), (stride, page * dim, dim, 1), storage_offset=2 * page * dim)
    g = gen(16)
    use = i32([[7, 1025, 3, 1099, 1024, 7], [7, 9, 1, 2, 0, 7]])[:, 1:5]
    n = 200
    seq = i32([0] * 100 + [1] * 100)
    at = torch.arange(100, dtype=torch.int32, device="cuda").repeat(2)
    kv = PagedKV(k_pool, v_pool)
    kvs = randn(g, n, 4, dim, kind="bf16")
    kv.append(kvs[:, :2], kvs[:, 2:], use, at, seq=seq)
    q = randn(g, 50, 12, dim, kind="bf16")[:, 2:10]
    hold = torch.full((50, 9, dim + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    out = hold[:, 1:9, :dim]
    first = i32([0, 30, 50])
    kv.attend_tree(q, use, i32([70, 80]), first, None, out=out)
    for r, (a, b, p) in enumerate(((0, 30, 70), (30, 50, 80))):
        keys = torch.arange(100, device="cuda")
        # only the pages in use as 64 bits
        ids = use[r].long()
        values = [x[ids].double() for x in (k_pool, v_pool)]
        want, _, tol, size, _, vmax = attention64(q[a:b], values, torch.arange(4, device="cuda"), keys, seen_by(None, a, b, keys, p), dim ** -0.5)
        close(out[a:b], want, bound_of(tol, size, vmax, want, "bf16", "bf16", wide=True))
    hold[:, 1:9, :dim] = 3.0
    assert bool((hold == 3.0).all())


@pytest.mark.parametrize("io,cache", TYPES)
def test_same_bits_captured_replayed_and_on_other_streams(io, cache):
    g, rng = gen(17), np.random.default_rng(17)
    c = Cache(g, 300, 2, 16, 128, cache)
    table = torch.from_numpy(rng.permutation(300).astype(np.int32).reshape(3, 100)).cuda()
    nodes = [40, 7, 64]
    lens, first = i32([900, 64, 1500]), i32(np.cumsum([0] + nodes))
    mask, _ = tree_mask([random_tree(rng, n) for n in nodes])
    q = randn(g, sum(nodes), 8, 128, kind=io)
    want = c.kv.attend_tree(q, table, lens, first, mask)
    for _ in range(3):
        assert torch.equal(c.kv.attend_tree(q, table, lens, first, mask), want)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    torch.cuda.synchronize()
    for st in streams:
        with torch.cuda.stream(st):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                out = c.kv.attend_tree(q, table, lens, first, mask)
        graphs.append((gr, out))
    torch.cuda.synchronize()
    for new_lens, new_nodes in (([1, 0, 700], [40, 7, 64]), ([1500, 1501, 20], [1, 100, 10]), ([1000, 3, 4], [0, 0, 111])):
        lens.copy_(i32(new_lens)), first.copy_(i32(np.cumsum([0] + new_nodes)))
        q.copy_(randn(g, sum(nodes), 8, 128, kind=io))
        want = c.kv.attend_tree(q, table, lens, first, mask)
        torch.cuda.synchronize()
        for st, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        # (a row of 1501 + 100 tokens is one longer than the table: NaN)
        assert all(torch.equal(out.nan_to_num(99.0), want.nan_to_num(99.0)) for _, out in graphs)


def test_refusals_and_calls_without_tokens():
    g = gen(20)
    c = Cache(g, 4, 2, 16, 64, "bf16")
    kv, table, lens, first = c.kv, torch.zeros(2, 2, dtype=torch.int32, device="cuda"), i32([3, 4]), i32([0, 2, 5])
    q = randn(g, 5, 4, 64, kind="bf16")
    mask = torch.zeros(5, 1, dtype=torch.int32, device="cuda")
    bad = [
        lambda: kv.attend_tree(q.half(), table, lens, first), lambda: kv.attend_tree(q, table, lens, first[:2]),
        lambda: kv.attend_tree(q, table, lens, first.long()), lambda: kv.attend_tree(q, table, lens[:1], first),
        lambda: kv.attend_tree(q, table, lens, first, mask[:4]), lambda: kv.attend_tree(q, table, lens, first, mask.bool()),
        lambda: kv.attend_tree(q, table, lens, first, mask[:, :0]), lambda: kv.attend_tree(q, table, lens, first, mask.cpu()),
        lambda: kv.attend_tree(q, table, lens, first, torch.zeros(5, 4, dtype=torch.int32, device="cuda")[:, ::2]),
        lambda: kv.attend_tree(q, table, lens, first, out=q[:4]), lambda: kv.attend_tree(q, table, lens, first, lse=torch.zeros(5, 3, device="cuda")),
        lambda: kv.commit(table, lens, i32([[0], [1], [2]])), lambda: kv.commit(table, lens, i32([[0], [1]]).long()),
        lambda: kv.commit(table, lens[:1], i32([[0], [1]])), lambda: kv.commit(table, lens, i32([[0], [1]]), new_lens=lens[:1]),
        lambda: kv.commit(table, lens, i32([[0, 1], [1, 2]]).t()), lambda: kv.commit(table, lens, i32([[0], [1]]).cpu()),
        lambda: tree_mask([[0]]), lambda: tree_mask([[-1, 1]]), lambda: tree_mask([[-2]]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for call, text in ((lambda: kv.attend_tree(q[:, :3], table, lens, first), "n_heads"), (lambda: kv.attend_tree(q, table, lens, first, scale=math.nan), "scale"),
                       (lambda: kv.attend_tree(q, table, lens, first, out=q[:1].expand(5, -1, -1)), "overlap"), (lambda: kv.commit(table, lens, i32([[0], [1]]), new_lens=lens), "new_lens")):
        with pytest.raises(Gpt2qError, match=text):
            call()
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    e = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert kv.attend_tree(e, table, lens, i32([0, 0, 0])).shape == (0, 4, 64)
    assert kv.attend_tree(e, table, lens, i32([0, 0, 0]), mask[:0]).shape == (0, 4, 64)
    assert kv.attend_tree(e, table[:0], none, i32([0])).shape == (0, 4, 64)
    assert kv.commit(table[:0], none, torch.empty(0, 3, dtype=torch.int32, device="cuda")).shape == (0,)
    assert torch.equal(kv.commit(table, lens, torch.empty(2, 0, dtype=torch.int32, device="cuda")), lens)
    m, d = tree_mask([[], [-1, 0, 0, 2, -1], []])
    assert m.flatten().tolist() == [1, 3, 5, 13, 16] and d.tolist() == [0, 1, 1, 2, 0]
    assert tree_mask([])[0].shape == (0, 1) and tree_mask([list(range(-1, 99))])[0][99].tolist() == [-1, -1, -1, 15]


# ------------------------------------------------------------------------------------- committing
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "i8", "e4m3"])
@pytest.mark.parametrize("kv,dim,page,layout", [(2, 64, 16, "hnd"), (12, 64, 5, "nhd"), (25, 256, 1, "hnd"), (1, 16, 64, "nhd")])
def test_commit(cache, kv, dim, page, layout):
    g, rng = gen(30), np.random.default_rng(30)
    nodes = [64, 1, 20, 5, 0, 40]
    lens = [70, 3, 0, 17, 9, -2]
    there = [max(0, p) + n for p, n in zip(lens, nodes)]
    pages = sum(-(-n // page) for n in there) + 1
    c = Cache(g, pages, kv, page, dim, cache, layout)
    table = tables(rng, there, page, pages)
    keep = [sorted(rng.permutation(64)[:30].tolist()), [0], list(range(20)), [], [], [0, 1, 2, 39]]
    accept = np.full((6, 33), -1, np.int32)
    for i, a in enumerate(keep):
        accept[i, :len(a)] = a
        accept[i, len(a) + 1:] = 3  # behind the end
    want = [[bits(p).clone() for p in c.pools], [None if s is None else s.clone() for s in c.scales]]
    t = table.cpu().numpy()
    for r, a in enumerate(keep):
        for i, x in enumerate(a):  # in order: sources are never behind their places
            s, d = max(0, lens[r]) + x, max(0, lens[r]) + i
            at, to = (int(t[r, s // page]), s % page), (int(t[r, d // page]), d % page)
            for p, f in zip(*want):
                p[to[0], :, to[1]] = p[at[0], :, at[1]]
                if f is not None:
                    f[to[0], :, to[1]] = f[at[0], :, at[1]]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    hold = i32(accept.repeat(2, 0))[::2]  # rows twice as far apart
    new = c.kv.commit(table, i32(lens), hold, status=status)
    assert int(status) == 0 and new.tolist() == [max(0, p) + len(a) for p, a in zip(lens, keep)]
    for p, f, wp, wf in zip(c.pools, c.scales, *want):
        assert torch.equal(bits(p), wp) and (f is None or torch.equal(f, wf))


@pytest.mark.parametrize("cache", ["bf16", "i8"])
def test_commit_stops_at_what_does_not_rise_or_has_no_page(cache):
    c = Cache(gen(31), 6, 1, 4, 64, cache)
    table = i32([[0, 1, -1, 2], [3, 9, 4, 5]])
    before = c.values[0].clone()

    def run(lens, accept):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        return c.kv.commit(table, i32(lens), i32(accept), status=status).tolist(), int(status)
    assert run([0, 0], [[0, 1, 1, 2], [0, -1, 0, 0]]) == ([2, 1], STATUS_POSITION)
    assert run([0, 0], [[3, 2, 0, 0], [-5, 0, 0, 0]])[0] == [1, 0]
    assert run([0, 0], [[0, 8, 9, -1], [3, 4, -1, -1]]) == ([1, 1], STATUS_PAGE)
    assert run([0, 0], [[12, 16, -1, -1], [2 ** 31 - 1, -1, -1, -1]]) == ([1, 0], STATUS_POSITION)
    assert run([13, 15], [[0, 2, 3, -1], [0, 1, -1, -1]]) == ([15, 16], STATUS_POSITION)
    assert before.shape == c.values[0].shape


@pytest.mark.parametrize("io,cache", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "i8"), ("f16", "e4m3")])
def test_steps_with_drafts_equal_steps_without(io, cache):
    """Three sequences decode with drafts: append at slots and depths, attention of the tree, commit; the cache afterwards and the accepted
    tokens' attention are those of a cache that took the accepted tokens one by one."""
    g, rng = gen(40), np.random.default_rng(40)
    kvh, heads, dim, page = 2, 8, 64, 8
    rows, total = 3, 64
    a, b = (Cache(gen(41), 30, kvh, page, dim, cache) for _ in range(2))
    table = tables(rng, [total] * rows, page, 30)
    rot = Rotary(dim)
    prompts = [5, 1, 17]
    seq = i32(np.repeat(np.arange(rows), prompts))
    pos = i32(np.concatenate([np.arange(p) for p in prompts]))
    k, v = (randn(g, sum(prompts), kvh, dim, kind=io) for _ in range(2))
    for c in (a, b):
        c.kv.append(k, v, table, pos, seq=seq, rotary=rot)
    lens = i32(prompts)
    for step in range(4):
        parents = [random_tree(rng, n) for n in (9, 1 + step, 30)]
        mask, depth = tree_mask(parents)
        nodes = [len(p) for p in parents]
        first = np.cumsum([0] + nodes)
        seq = i32(np.repeat(np.arange(rows), nodes))
        node = i32(np.concatenate([np.arange(n) for n in nodes]))
        k, v, q = (randn(g, int(first[-1]), h, dim, kind=io) for h in (kvh, kvh, heads))
        base = lens[seq.long()]
        turned = a.kv.append(k, v, table, base + depth, seq=seq, rotary=rot, q=q, slot=base + node)
        out = a.kv.attend_tree(turned, table, lens, i32(first), mask)
        accept = np.full((rows, 6), -1, np.int32)
        for r, p in enumerate(parents):
            path, at = [], int(rng.integers(0, len(p)))
            while at >= 0:
                path.append(at)
                at = p[at]
            path = path[::-1][:6]
            accept[r, :len(path)] = path
            for i, x in enumerate(path):  # one by one
                t = int(first[r]) + x
                one = slice(t, t + 1)
                at = lens[r:r + 1] + i
                qt = b.kv.append(k[one], v[one], table[r:r + 1], at, rotary=rot, q=q[one])
                assert torch.equal(qt, turned[one])
                o = b.kv.attend(qt, table[r:r + 1], at + 1)
                e = torch.finfo(T[io]).eps
                # two roundings of the output, of weights to 16 bits (2^-9 of |v| < 8 at the most), and of sums in another order
                err = (o.double() - out[one].double()).abs()
                assert bool((err <= o.double().abs() * e + (2.0 ** -5 if io != "f32" else 2.0 ** -15)).all()), float(err.max())
        lens = a.kv.commit(table, lens, i32(accept))
    for r in range(rows):
        n = int(lens[r])
        at = torch.arange(n, dtype=torch.int32, device="cuda")
        s = torch.full((n,), r, dtype=torch.int32, device="cuda")
        x, y = a.kv.read(table, at, seq=s, dtype=torch.float32), b.kv.read(table, at, seq=s, dtype=torch.float32)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_commit_of_long_lists(cache):
    """Lists of several hundred tokens, that end at and around a block's 256, at the width and at a token that does not rise."""
    g, rng = gen(32), np.random.default_rng(32)
    nodes, page = 700, 16
    ends = [255, 256, 257, 511, 512, 513, 600, 300]
    c = Cache(g, 420, 2, page, 32, cache)
    table = tables(rng, [nodes + 100] * 8, page, 420)
    accept = np.full((8, 600), -1, np.int32)
    for r, n in enumerate(ends):
        accept[r, :n] = np.sort(rng.permutation(nodes)[:n])
    accept[7, 290] = accept[7, 289]  # ends there
    ends[7] = 290
    want = [bits(p).clone() for p in c.pools]
    t = table.cpu().numpy()
    for r, n in enumerate(ends):
        src = 50 + accept[r, :n]
        dst = 50 + np.arange(n)
        at = torch.as_tensor(t[r, src // page]).long().cuda(), torch.as_tensor(src % page).cuda()
        to = torch.as_tensor(t[r, dst // page]).long().cuda(), torch.as_tensor(dst % page).cuda()
        for p, w in zip(c.pools, want):
            w[to[0], :, to[1]] = bits(p)[at[0], :, at[1]].clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    new = c.kv.commit(table, torch.full((8,), 50, dtype=torch.int32, device="cuda"), i32(accept), status=status)
    assert new.tolist() == [50 + n for n in ends] and int(status) == STATUS_POSITION
    for p, w in zip(c.pools, want):
        assert torch.equal(bits(p), w)
