"""Drafted tokens behind a prefix whose values hold an infinity or a NaN: every token sees the prefix, so it has its way in that one
element of the head, wherever the entry lies, and the other elements are as without it."""
import math

import numpy as np
import pytest
import torch

from smelt_b200.paged import tree_mask

from .paged_oracle import Cache, gen, randn, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


@pytest.mark.parametrize("io,cache", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "e4m3"), ("bf16", "e4m3"),
                                      ("f16", "e4m3")])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("n", [2, 80])
def test_a_prefix_with_an_infinity(io, cache, page, n):
    g, rng = gen(1), np.random.default_rng(1)
    prefix, dim, at = 37, 64, 3
    pages = -(-(prefix + n) // page) + 1
    c = Cache(g, pages, 2, page, dim, cache)
    table = tables(rng, [prefix + n], page, pages)
    mask, _ = tree_mask([[-1] + [int(rng.integers(-1, i)) for i in range(1, n)]])
    q = randn(g, n, 4, dim, kind=io, scale=0.1)  # every key has a weight
    lens, first = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([prefix], [0, n]))
    others = torch.arange(dim, device="cuda") != at
    for chain in (False, True):
        args = q, table, lens, first, None if chain else mask
        lse, other = (torch.empty(n, 4, device="cuda") for _ in range(2))
        clean = c.kv.attend_tree(*args, lse=lse)
        for pos in (36, 32, 3):
            entry = c.pools[1][table[0, pos // page].item(), :, pos % page]
            for what in (math.inf, math.nan):
                hold = entry.clone()
                if cache == "e4m3":
                    entry.view(torch.int8)[:, at] = 0x7f  # NaN; there is no infinity
                else:
                    entry[:, at] = what
                out = c.kv.attend_tree(*args, lse=other)
                assert not bool(torch.isfinite(out[..., at]).any()), (pos, what)
                assert torch.equal(out[..., others], clean[..., others]) and torch.equal(other, lse), (pos, what)
                entry.copy_(hold)
