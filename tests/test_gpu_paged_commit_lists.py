"""Lists of accepted tokens that gpt2q_commit_paged refuses: no layer's cache is touched."""
import numpy as np
import pytest
import torch

from smelt_b200._ffi import Gpt2qError
from smelt_b200.gpu import Gpu
from smelt_b200.paged import PagedKV

from .helpers import TINY, make_pack

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def test_lists_that_do_not_rise_or_leave_the_table():
    hd = TINY.n_embd // TINY.n_head
    layers = [PagedKV(*(torch.randn(8, TINY.n_head, 16, hd, device="cuda") for _ in range(2))) for _ in range(TINY.n_layer)]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    with Gpu(make_pack(TINY, "auto"), max_tokens=16) as g:
        hold = [x.clone() for kv in layers for x in (kv.k, kv.v)]
        for lens, accept, text in (([3, 5], [[1, 3], [0, 2, 2]], "rise"), ([3, 5], [[4, 3], [1]], "rise"), ([3, 5], [[1], [2, 59]], "past the table"),
                                   ([64, 0], [[0], [1]], "past the table")):
            with pytest.raises(Gpt2qError, match=text):
                g.commit_paged(lens, accept, layers, table)
            assert all(torch.equal(x, y) for x, y in zip(hold, (x for kv in layers for x in (kv.k, kv.v))))
        assert g.commit_paged([3, 5], [[1, 3], [2, 58]], layers, table).tolist() == [5, 7]
        assert torch.equal(layers[0].k[0, :, 3], hold[0][0, :, 4]) and torch.equal(layers[-1].v[4, :, 6], hold[-1][7, :, 15])
