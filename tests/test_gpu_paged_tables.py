"""Page tables that the model's paged calls refuse: before anything is written."""
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


def caches(pages, page):
    hd = TINY.n_embd // TINY.n_head
    return [PagedKV(*(torch.full((pages, TINY.n_head, page, hd), 7.0, device="cuda") for _ in range(2))) for _ in range(TINY.n_layer)]


def untouched(layers):
    return all(bool((x == 7.0).all()) for kv in layers for x in (kv.k, kv.v))


def test_rows_that_share_storage_are_refused():
    """Several new tokens of one sequence as rows of one expanded table row, and overlapping windows of a table."""
    with Gpu(make_pack(TINY, "auto"), max_seqs=2) as g:
        g.prefill([np.arange(5, dtype=np.uint32)])
        one = torch.arange(4, dtype=torch.int32, device="cuda")[None]
        flat = torch.arange(16, dtype=torch.int32, device="cuda") % 8
        for table in (one.expand(3, -1), flat.as_strided((3, 4), (2, 1))):
            layers = caches(8, 16)
            with pytest.raises(Gpt2qError, match="page table"):
                g.decode_paged([1, 2, 3], [0, 1, 2], layers, table)
            for row in (0, 1, 2):
                with pytest.raises(Gpt2qError, match="page table"):
                    g.page_out(0, 5, layers, table, row)
            assert untouched(layers)
        # the same rows, each with its own storage
        layers = caches(8, 16)
        g.page_out(0, 5, layers, one.expand(3, -1).contiguous(), 2)
        assert not untouched(layers)
        assert g.decode_paged([1], [5], layers, one[:, :4]).shape == (1,)
