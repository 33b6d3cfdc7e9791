"""A drafted token whose value is NaN, with a score so low that its weight is 0: those that see it give NaN all the same, as 0 times NaN
does, and the others are as without it."""
import math

import numpy as np
import pytest
import torch

from .paged_oracle import Cache, gen, randn, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


@pytest.mark.parametrize("io,cache", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "i8"), ("bf16", "i8"),
                                      ("f16", "e4m3"), ("f32", "e4m3")])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("n", [2, 60])
def test_a_weight_of_nothing(io, cache, page, n):
    g, rng = gen(1), np.random.default_rng(1)
    prefix, dim = 20, 64
    pages = -(-(prefix + n) // page) + 1
    c = Cache(g, pages, 1, page, dim, cache)
    table = tables(rng, [prefix + n], page, pages)
    q = randn(g, n, 4, dim, kind=io).abs()
    node = n - 2
    at = table[0, (prefix + node) // page].item(), 0, (prefix + node) % page
    # a key opposite to all queries: scores about 1000 below the others
    if cache in ("i8", "e4m3"):
        c.pools[0][at] = torch.full((dim,), -64.0, device="cuda").to(c.pools[0].dtype)
        c.scales[0][at] = 4.0
    else:
        c.pools[0][at] = -200.0
    mask = torch.full((n, (n + 31) // 32), 0, dtype=torch.int64)
    for t in range(n):
        for j in {t, node} if t % 2 == node % 2 else {t}:
            mask[t, j // 32] |= 1 << (j % 32)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32).cuda()
    args = q, table, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([prefix], [0, n])), mask
    clean = c.kv.attend_tree(*args)
    assert bool(torch.isfinite(clean).all())
    if cache == "i8":
        c.scales[1][at] = math.nan
    elif cache == "e4m3":
        c.pools[1].view(torch.int8)[(*at, 5)] = 0x7f
    else:
        c.pools[1][(*at, 5)] = math.nan
    out = c.kv.attend_tree(*args)
    sees = torch.arange(n, device="cuda") % 2 == node % 2
    assert bool(torch.isnan(out[sees]).flatten(1).any(1).all())
    assert torch.equal(out[~sees], clean[~sees])
