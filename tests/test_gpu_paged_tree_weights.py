"""What the rounding of weights to 16 bits leaves in results on wide tiles: nothing where all keys have one scale, or a token sees
one key.

Weights times scales are rounded to 11 bits, relative to 2^-11 at the most, and corrected by the quotient of their sums before
and after. Where all weights times scales are equal, or there is one, only fp32 operations are left: 2^-20 covers the quotient, which
goes by way of numbers of 8 bits (2^-8 of up to 2^-11, twice: 2^-18), so 2^-17 in all, and then the output's own rounding."""
import numpy as np
import pytest
import torch

from smelt_b200.paged import PagedKV

from .paged_oracle import T, close, gen, quantise, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("io", ["f16", "bf16"])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("prefix,n,heads", [(0, 20, 4), (100, 30, 4), (5000, 64, 8), (40000, 12, 2)])
def test_one_scale_for_all(io, cache, prefix, n, heads):
    """Scores of 0 over entries of one scale that 11 bits do not hold: the mean of the values."""
    g = gen(1)
    page, dim = 64, 64
    pages = -(-(prefix + n) // page)
    for scale in (1 / 126, 1 / 127.3, 0.0123456):
        codes = [quantise(randn(g, pages, 1, page, dim), cache)[0] for _ in range(2)]
        scales = [torch.full((pages, 1, page), scale, device="cuda") for _ in range(2)]
        kv = PagedKV(*codes, *scales)
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        q = torch.zeros(n, heads, dim, dtype=T[io], device="cuda")
        out = kv.attend_tree(q, table, i32([prefix]), i32([0, n]))
        v = codes[1].double().view(-1, dim) * scales[1][0, 0, 0].double()
        mean = (v.cumsum(0) / torch.arange(1, len(v) + 1, device="cuda")[:, None])[prefix:prefix + n]
        size = (v.abs().cumsum(0) / torch.arange(1, len(v) + 1, device="cuda")[:, None])[prefix:prefix + n]
        # sums of up to 40 thousand terms in fp32, each rounded by 2^-23 of the sum of magnitudes at the most, 16 keys at a time
        tol = mean.abs() * (torch.finfo(T[io]).eps / 2) * 1.01 + size * (2.0 ** -17 + (prefix + n) / 16 * 2.0 ** -23) + (2.0 ** -25 if io == "f16" else 0)
        close(out, mean[:, None].expand(-1, heads, -1), tol[:, None], scale)


@pytest.mark.parametrize("io", ["f16", "bf16"])
@pytest.mark.parametrize("cache", ["f16", "bf16", "i8", "e4m3"])
def test_a_token_that_sees_one_key_gives_its_value(io, cache):
    if cache in ("f16", "bf16") and cache != io:
        pytest.skip("16-bit caches take their own type")
    from .paged_oracle import Cache

    g = gen(2)
    n, heads, dim = 40, 4, 128
    c = Cache(g, 3, 1, 16, dim, cache)
    table = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    q = randn(g, n, heads, dim, kind=io)
    mask = torch.zeros(n, 2, dtype=torch.int64)
    for t in range(n):  # each one itself
        mask[t, t // 32] = 1 << (t % 32)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32).cuda()
    out = c.kv.attend_tree(q, table, i32([0]), i32([0, n]), mask)
    v = c.values[1].transpose(1, 2).reshape(48, dim)[:n][:, None].expand(-1, heads, -1)
    if cache == io:
        assert torch.equal(out, v.to(T[io]))
    close(out, v, v.abs() * (torch.finfo(T[io]).eps / 2 * 1.01 + 2.0 ** -17) + (2.0 ** -25 if io == "f16" else 0))
