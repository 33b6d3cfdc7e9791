"""Integers of drafted tokens' calls that 32 bits do not hold."""
import numpy as np
import pytest
import torch

from smelt_b200.gpu import Gpu, _int32
from smelt_b200.paged import PagedKV

from .helpers import TINY, make_pack


def test_numbers_that_do_not_fit():
    for x in ([2 ** 31], [-2 ** 31 - 1], np.array([1, 2 ** 40]), [0, 2 ** 32]):
        with pytest.raises(ValueError, match="what"):
            _int32(x, "what")
    assert _int32([2 ** 31 - 1, -2 ** 31], "what").tolist() == [2 ** 31 - 1, -2 ** 31] and _int32([], "what").size == 0


@pytest.mark.gpu
def test_calls():
    hd = TINY.n_embd // TINY.n_head
    layers = [PagedKV(*(torch.zeros(8, TINY.n_head, 16, hd, device="cuda") for _ in range(2))) for _ in range(TINY.n_layer)]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    with Gpu(make_pack(TINY, "auto"), max_tokens=16) as g:
        tok = [np.array([1, 2], np.uint32), np.array([3], np.uint32)]
        for parents, lens, text in (([[-1, 2 ** 32], [-1]], [0, 0], "parents"), ([[-1, 2 ** 32 - 1], [-1]], [0, 0], "parents"),
                                    ([[-1, 0], [-1]], np.array([2 ** 32, 0]), "lens")):
            with pytest.raises(ValueError, match=text):
                g.verify_paged(tok, parents, lens, layers, table)
        with pytest.raises(ValueError, match="accept"):
            g.commit_paged([0, 0], [np.array([2 ** 32 + 1]), []], layers, table)
        with pytest.raises(ValueError, match="lens"):
            g.commit_paged(np.array([2 ** 33, 0]), [[0], [0]], layers, table)
        assert [len(x) for x in g.verify_paged(tok, [[-1, 0], [-1]], [0, 0], layers, table)] == [2, 1]
