"""A `first` that names every token once for each of many rows: the work it asks for is not begun."""
import pytest
import torch

from smelt_b200.paged import STATUS_POSITION

from .paged_oracle import T, Cache, gen, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


@pytest.mark.parametrize("io,cache", [("bf16", "bf16"), ("f16", "i8"), ("f32", "i8"), ("f32", "f16"), ("f32", "f32")])
def test_tokens_that_are_named_again_and_again(io, cache):
    g = gen(1)
    rows, n, heads = 64, 512, 4
    c = Cache(g, 40, 1, 16, 64, cache)
    table = torch.arange(40, dtype=torch.int32, device="cuda").expand(rows, 40).contiguous()
    q = randn(g, n, heads, 64, kind=io)
    out = torch.full((n, heads, 64), 5.0, dtype=T[io], device="cuda")
    lse = torch.full((n, heads), 5.0, device="cuda")
    lens = torch.full((rows,), 20, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    again = torch.tensor([0, n] * (rows // 2) + [0], dtype=torch.int32, device="cuda")
    c.kv.attend_tree(q, table, lens, again, None, out=out, lse=lse, status=status)
    assert int(status) == STATUS_POSITION and bool((out == 5.0).all()) and bool((lse == 5.0).all())
    # every token once, in the same call otherwise
    once = torch.tensor([n * r // rows for r in range(rows + 1)], dtype=torch.int32, device="cuda")
    status.zero_()
    c.kv.attend_tree(q, table, lens, once, None, out=out, lse=lse, status=status)
    assert int(status) == 0 and not bool((lse == 5.0).any())
