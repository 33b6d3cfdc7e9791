"""Drafted tokens over 8-bit caches whose values' scales differ by many powers of two: a scale that a token does not see leaves its
result as it was, to the bit, and what it does see is right relative to the largest value that it sees.

The bound is that of paged_oracle.py with the largest |v| over the keys that a token sees. Weights times scales are held in fp16
relative to the largest scale seen: on the warp-level kernel times 2^10 in two pieces (2^-35 of it per key, which the bound has), on
wide tiles times 2^6 in one, where half a step of the smallest numbers is 2^-25: 2^-31 of it per key."""
import math

import numpy as np
import pytest
import torch

from smelt_b200.paged import tree_mask

from .paged_oracle import T, U, WEIGHT, Cache, attention64, bound_of, close, gen, randn, tables

pytestmark = pytest.mark.gpu
# page, dim, drafted tokens, heads, kv heads, prefix
SHAPES = [(16, 64, 80, 8, 2, 37), (5, 64, 80, 8, 2, 37), (16, 128, 150, 8, 2, 200), (16, 128, 20, 4, 2, 150), (16, 256, 9, 2, 2, 3), (32, 80, 30, 6, 1, 0),
          (64, 128, 300, 16, 1, 1000)]


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


class Tree:
    """One row of `n` drafted tokens in a random tree behind a prefix."""

    def __init__(self, seed, page, dim, n, heads, kv, prefix, io, cache, sizes=0.5):
        g, rng = gen(seed), np.random.default_rng(seed)
        self.n, self.prefix, self.page, self.io, self.dim = n, prefix, page, io, dim
        pages = -(-(prefix + n) // page) + 1
        self.c = Cache(g, pages, kv, page, dim, cache, sizes=sizes)
        self.table = tables(rng, [prefix + n], page, pages)
        self.mask, _ = tree_mask([[-1 if rng.random() < 0.1 else int(rng.integers(max(-1, i - 6), i)) for i in range(n)]])
        words = self.mask.cpu().numpy().view(np.uint32)
        self.sees = torch.tensor([[bool(words[t, j // 32] >> (j % 32) & 1) for j in range(n)] for t in range(n)], device="cuda")
        self.q = randn(g, n, heads, dim, kind=io)
        # the rule by which the calls take wide tiles
        self.wide = io != "f32" and dim <= 128 and page % 8 == 0 and n * (heads // kv) > 8

    def scale_at(self, node):
        at = self.prefix + node
        return self.c.scales[1][self.table[0, at // self.page].item(), :, at % self.page]

    def attend(self):
        lse = torch.empty(self.q.shape[:2], device="cuda")
        return self.c.kv.attend_tree(self.q, self.table, i32([self.prefix]), i32([0, self.n]), self.mask, lse=lse), lse

    def check(self, tokens, out, lse):
        values, cache = self.c.values, self.c.kind
        for t in tokens:
            keys = torch.cat([torch.arange(self.prefix, device="cuda"), self.prefix + self.sees[t].nonzero()[:, 0]])
            seen = torch.ones(1, len(keys), dtype=torch.bool, device="cuda")
            want, wl, tol, size, rel, vmax = attention64(self.q[t:t + 1], values, self.table[0], keys, seen, self.dim ** -0.5)
            tol = bound_of(tol, size, vmax, want, self.io, cache, wide=self.wide) + (len(keys) * 2.0 ** -31 * vmax if self.wide else 0)
            close(out[t:t + 1], want, tol, ("out", t))
            close(lse[t:t + 1], wl, rel + (wl.abs() + 1) * 4 * U + 2.0 ** -20 + (1.01 * WEIGHT[0] if self.wide else 0), ("lse", t))


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_scale_that_is_not_seen_changes_nothing(shape, io, cache):
    x = Tree(1, *shape, io, cache)
    clean, lse = x.attend()
    assert bool(torch.isfinite(clean).all())
    x.check(range(x.n), clean, lse)
    nodes = [1, x.n // 2, x.n - 2, x.n - 1]
    for chosen in ([nodes[0]], [nodes[1]], [nodes[2]], nodes):
        for factor in (2.0 ** 20, 2.0 ** 40, 1e30):
            hold = [x.scale_at(i).clone() for i in chosen]
            for i in chosen:
                x.scale_at(i).mul_(factor)
            out, other = x.attend()
            seers = x.sees[:, chosen].any(1)
            assert torch.equal(out[~seers], clean[~seers]), (chosen, factor, float((out[~seers].double() - clean[~seers].double()).abs().max()))
            assert torch.equal(other, lse)
            if io != "f16":  # (whose largest number they are past)
                x.check(seers.nonzero()[:, 0].tolist(), out, other)
            for i, h in zip(chosen, hold):
                x.scale_at(i).copy_(h)


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("sizes", [4.0, 9.0])
def test_results_are_right_relative_to_what_is_seen(shape, io, cache, sizes):
    """Scales over e^(+-3 sizes), with queries that leave most scores of order one."""
    x = Tree(2, *shape, io, cache, sizes)
    x.q.mul_(1e-3 * math.exp(-2 * sizes))
    x.check(range(x.n), *x.attend())


@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,prefix", [(5, 100), (16, 100), (16, 250)])
def test_a_chain_whose_scales_rise(io, page, prefix):
    """Without a mask: every drafted token's values are 2^9 times those of the one before."""
    n = 12
    x = Tree(3, page, 64, n, 4, 2, prefix, io, "i8")
    x.mask = None
    x.sees = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    for i in range(n):
        x.scale_at(i).fill_(2.0 ** (9 * i - 30))
    # (2^6 * 127 is the largest that fp16 has)
    x.check(range(n if io != "f16" else 5), *x.attend())


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_scales_of_either_sign_and_of_zero(shape, io, cache):
    """(append writes none that are negative, but a scale is any number)"""
    x = Tree(4, *shape, io, cache)
    g = gen(5)
    for s in x.c.scales:
        sign = torch.randint(-1, 2, s.shape, device="cuda", generator=g).float()
        s.mul_(sign)
    x.check(range(x.n), *x.attend())
