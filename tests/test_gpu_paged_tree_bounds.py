"""Attention of drafted tokens where the warp-level kernel has it, within the bound of weights in two or three 16-bit pieces
(paged_oracle.py), batches of uneven drafts around the rule that chooses the kernel, and what a commit that ends early moves."""
import numpy as np
import pytest
import torch

from smelt_b200.paged import STATUS_PAGE, STATUS_POSITION, tree_mask

from .paged_oracle import T, U, Cache, attention64, bound_of, close, gen, randn, tables

pytestmark = pytest.mark.gpu
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "i8"), ("bf16", "i8"), ("f16", "i8"),
         ("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e4m3")]


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def check(seed, prefixes, nodes, heads, kv, dim, io, cache, page, chain):
    g, rng = gen(seed), np.random.default_rng(seed)
    there = [p + n if n else 0 for p, n in zip(prefixes, nodes)]
    pages = sum(-(-n // page) for n in there) + 1
    c = Cache(g, pages, kv, page, dim, cache)
    table = tables(rng, there, page, pages)
    first = np.cumsum([0] + nodes)
    mask, _ = tree_mask([[-1 if rng.random() < 0.1 else int(rng.integers(max(-1, i - 6), i)) for i in range(n)] for n in nodes])
    q = randn(g, int(first[-1]), heads, dim, kind=io)
    lse = torch.empty(int(first[-1]), heads, device="cuda")
    out = c.kv.attend_tree(q, table, i32(prefixes), i32(first), None if chain else mask, lse=lse)
    # the rule by which a call takes wide tiles
    wide = io != "f32" and cache != "f32" and dim <= 128 and page % 8 == 0 and sum(nodes) * (heads // kv) > 8 * len(nodes)
    for r, (p, n) in enumerate(zip(prefixes, nodes)):
        a, b = int(first[r]), int(first[r + 1])
        if a == b:
            continue
        keys = torch.arange(p + n, device="cuda")
        own = keys - p
        if chain:
            seen = own[None] <= torch.arange(n, device="cuda")[:, None]
        else:
            j = own.clamp(min=0)
            seen = (own < 0)[None] | ((mask[a:b].long()[:, j // 32] >> (j % 32)) & 1 == 1)
        want, wl, tol, size, rel, vmax = attention64(q[a:b], c.values, table[r], keys, seen, dim ** -0.5)
        close(out[a:b], want, bound_of(tol, size, vmax, want, io, cache, wide=wide), ("out", r))
        if not wide:
            close(lse[a:b], wl, rel + (wl.abs() + 1) * 4 * U + 2.0 ** -20, ("lse", r))
    return wide


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("prefixes,nodes,heads,kv,dim,page", [
    ([33, 200, 5], [2, 1, 3], 12, 12, 64, 16), ([1000, 17], [1, 1], 16, 2, 128, 64), ([70, 31], [33, 9], 6, 2, 192, 16), ([300], [70], 8, 2, 64, 5),
    ([3000, 0], [40, 7], 4, 1, 256, 24)])
def test_warp_level(io, cache, prefixes, nodes, heads, kv, dim, page, chain):
    assert not check(1, prefixes, nodes, heads, kv, dim, io, cache, page, chain)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("nodes", [[100] + [0] * 63, [100] + [1] * 28 + [0] * 35, [101] + [1] * 28 + [0] * 35, [1] * 30 + [300] + [2] * 20 + [0] * 5])
def test_uneven_drafts(io, cache, nodes):
    """One long draft among rows of one token or none: on either side of the rule, with four query heads to a kv head."""
    rng = np.random.default_rng(3)
    check(2, [int(x) for x in rng.integers(0, 700, len(nodes))], nodes, 8, 2, 64, io, cache, 16, False)


@pytest.mark.parametrize("cache", ["f32", "bf16", "i8", "e4m3"])
def test_what_a_commit_that_ends_early_moves(cache):
    """The list's beginning, codes and scales, and nothing behind it."""
    def bits(x):
        return x.view(torch.int8) if x.element_size() == 1 else x

    table = i32([[0, 1, -1, 2], [3, 9, 4, 5]])
    for lens, accept, kept, bit in (
            ([0, 0], [[0, 1, 1, 2], [0, -1, 0, 0]], [2, 1], STATUS_POSITION), ([0, 0], [[3, 2, 0, 0], [-5, 0, 0, 0]], [1, 0], STATUS_POSITION),
            ([0, 0], [[0, 8, 9, -1], [3, 4, -1, -1]], [1, 1], STATUS_PAGE), ([0, 0], [[12, 16, -1, -1], [2 ** 31 - 1, -1, -1, -1]], [1, 0], STATUS_POSITION),
            ([2, 1], [[1, 3, 5, 4], [2, 5, -1, 0]], [3, 1], STATUS_POSITION | STATUS_PAGE), ([13, 15], [[0, 2, 3, -1], [0, 1, -1, -1]], [2, 1], STATUS_POSITION)):
        c = Cache(gen(31), 6, 2, 4, 64, cache)
        want = [bits(p).clone() for p in c.pools] + [s.clone() for s in c.scales if s is not None]
        t = table.cpu().numpy()
        for r in range(2):
            for i in range(kept[r]):
                s, d = lens[r] + accept[r][i], lens[r] + i
                for w in want:
                    w[int(t[r, d // 4]), :, d % 4] = w[int(t[r, s // 4]), :, s % 4]
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        new = c.kv.commit(table, i32(lens), i32(accept), status=status)
        assert new.tolist() == [n + k for n, k in zip(lens, kept)] and int(status) == bit, (lens, accept, new.tolist(), int(status))
        got = [bits(p) for p in c.pools] + [s for s in c.scales if s is not None]
        assert all(torch.equal(x, y) for x, y in zip(got, want)), (lens, accept)
