"""Drafted tokens over a table of 2^31 positions (128 entries of 2^24 tokens, which are all the same page)."""
import numpy as np
import pytest
import torch

from smelt_b200.paged import STATUS_POSITION, PagedKV

from .paged_oracle import attention64, bound_of, close, gen, randn

pytestmark = pytest.mark.gpu
PAGE, DIM = 1 << 24, 16


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("io", ["bf16", "f32"])  # wide tiles, warp-level kernel
def test_a_row_past_the_longest_beside_others(io):
    g = gen(1)
    k, v = (randn(g, 1, 1, PAGE, DIM, kind="bf16") for _ in range(2))
    kv = PagedKV(k, v)
    values = [x[:, :, :256].double() for x in (k, v)]
    table = torch.zeros(3, 128, dtype=torch.int32, device="cuda")
    n, heads = 9, 4
    q = randn(g, 3 * n, heads, DIM, kind=io)
    for over in (2 ** 31 - 1, 2 ** 31 - 70, 2 ** 31 - 4096):
        lens = [100, over, 30]
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lse = torch.empty(3 * n, heads, device="cuda")
        out = kv.attend_tree(q, table, i32(lens), i32([0, n, 2 * n, 3 * n]), lse=lse, status=status)
        assert int(status) == STATUS_POSITION
        assert bool(torch.isnan(out[n:2 * n]).all()) and bool(torch.isnan(lse[n:2 * n]).all())
        for r in (0, 2):
            keys = torch.arange(lens[r] + n, device="cuda")
            seen = keys[None] <= lens[r] + torch.arange(n, device="cuda")[:, None]
            a = slice(r * n, (r + 1) * n)
            want, wl, tol, size, _, vmax = attention64(q[a], values, torch.zeros(1, dtype=torch.int64, device="cuda").expand(1), keys, seen, DIM ** -0.5)
            close(out[a], want, bound_of(tol, size, vmax, want, io, "bf16", wide=True), (over, r))
            assert bool(torch.isfinite(lse[a]).all())
