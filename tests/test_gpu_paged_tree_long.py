"""Drafted tokens behind so many keys that a block has more of a row than its products are summed over in TMEM: rows that share
their pages, one block or more each.

Where all weights are equal and the values of one sign, what is left is the sums' own error. 128 tiles of 128 keys, 16 keys at a time,
are 1024 additions that each round a running sum towards zero, by half a unit of its last place on average: 2^-24 of the final sum
at the most, 2^-14 in all. The outputs' own rounding averages out over 128 dims whose means are evenly spread over one step of the type
to half a step over the number of dims, 2^-10 / 2 / 128, and not worse than 2^-14 with uneven spreading."""
import numpy as np
import pytest
import torch

from smelt_b200.paged import PagedKV

from .paged_oracle import T, Cache, attention64, bound_of, close, gen, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("cache", ["f16", "i8"])
@pytest.mark.parametrize("n,tokens", [(131072, 16), (65536, 150)])
def test_a_running_sum_of_one_sign(cache, n, tokens):
    dim, page, rows = 128, 1024, 160
    share = torch.arange(dim, device="cuda").double() / dim
    j = torch.arange(n, device="cuda")
    high = (j[:, None] * 0.6180339887498949) % 1.0 < share[None]  # of the keys, evenly
    if cache == "f16":
        # full significands: a product's bits do not fit the sum
        v = torch.where(high, 1.3330078125, 1.33203125).half().view(n // page, 1, page, dim)
        kv, values = PagedKV(torch.zeros_like(v), v), v.double()
    else:
        v = torch.where(high, 127, 126).to(torch.int8).view(n // page, 1, page, dim)
        s = torch.full((n // page, 1, page), 1 / 126, device="cuda")
        kv, values = PagedKV(torch.zeros_like(v), v, s, s.clone()), v.double() * s.double()[..., None]
    want = values.view(n, dim).mean(0)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(rows, -1).contiguous()
    q = torch.zeros(rows * tokens, 1, dim, dtype=torch.float16, device="cuda")
    words = (tokens + 31) // 32
    mask = torch.full((rows * tokens, words), -1, dtype=torch.int32, device="cuda")
    out = kv.attend_tree(q, table, torch.full((rows,), n - tokens, dtype=torch.int32, device="cuda"), i32(np.arange(rows + 1) * tokens), mask)
    rel = (out[:, 0].double() / want - 1).view(rows, tokens, dim).mean((1, 2))
    assert float(rel.abs().max()) <= 2.0 ** -14 + 2.0 ** -14, float(rel.abs().max())


@pytest.mark.parametrize("io,cache", [("f16", "f16"), ("bf16", "bf16"), ("f16", "i8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("tokens,heads,dim", [(6, 4, 128), (40, 4, 128), (70, 2, 64)])
@pytest.mark.parametrize("rise", [False, True])
def test_sums_in_memory(io, cache, tokens, heads, dim, rise):
    """Scores and values that rise with the position: the reference of the weights, and of the values' scales, moves all the time."""
    g = gen(1)
    page, rows = 64, 160
    prefix = 70001
    total = prefix + tokens
    pages = -(-total // page)
    c = Cache(g, pages, 1, page, dim, cache, sizes=0.0 if rise else 0.5)
    if rise:
        up = torch.linspace(0.0, 1.0, pages * page, device="cuda").view(pages, 1, page)
        # keys along one direction, with scores from 0 to 30 for queries of all ones; values from 1 to 2^10 times as large
        if cache in ("i8", "e4m3"):
            c.pools[0].copy_(torch.ones_like(c.pools[0].float()).to(c.pools[0].dtype))
            c.scales[0].copy_(up * 30)
            c.scales[1].mul_(2.0 ** (10 * up.round(decimals=2)))
        else:
            c.pools[0].copy_((up * 30)[..., None].expand(-1, -1, -1, dim).to(T[cache]))
            c.pools[1].mul_((2.0 ** (6 * up))[..., None].to(T[cache]))
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(rows, -1).contiguous()
    q = randn(g, rows * tokens, heads, dim, kind=io)
    if rise:
        q.fill_(1.0 / dim)
    lse = torch.empty(rows * tokens, heads, device="cuda")
    sm = 1.0 if rise else dim ** -0.5
    out = c.kv.attend_tree(q, table, torch.full((rows,), prefix, dtype=torch.int32, device="cuda"), i32(np.arange(rows + 1) * tokens), None, scale=sm, lse=lse)
    values = c.values
    keys = torch.arange(total, device="cuda")
    seen = keys[None] <= prefix + torch.arange(tokens, device="cuda")[:, None]
    for r in (0, 77, 159):
        a = slice(r * tokens, (r + 1) * tokens)
        want, wl, tol, size, rel, vmax = attention64(q[a], values, table[r], keys, seen, sm)
        e = bound_of(tol, size, vmax, want, io, cache, wide=True)
        close(out[a], want, e, r)
        # sums in TMEM: 1024 additions of up to 2^-23 of a sum of magnitudes, and those in memory
        e = want.abs() * (torch.finfo(T[io]).eps / 2) + size * (2.0 ** -13 + 2 * (2.0 ** -8 if cache == "bf16" else 2.0 ** -11)) + vmax * 2.0 ** -16
        close(out[a], want, e, ("tight", r))
