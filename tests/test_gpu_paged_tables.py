"""Page tables that the model's paged calls refuse: before anything is written."""
import ctypes as C

import numpy as np
import pytest
import torch

from smelt_b200 import _ffi
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


@pytest.mark.parametrize("change", [dict(ids=None), dict(width=0), dict(ld=3), dict(ld=-4)])
def test_bad_tables_are_refused_whatever_the_row(change):
    with Gpu(make_pack(TINY, "auto"), max_seqs=2) as g:
        g.prefill([np.arange(5, dtype=np.uint32)])
        ids = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
        layers = caches(8, 16)
        arr = (_ffi.PagedKV * len(layers))(*(kv.c for kv in layers))
        t = _ffi.PageTable(**(dict(ids=ids.data_ptr(), n_rows=3, width=4, ld=4) | change))
        torch.cuda.synchronize()
        tok, pos = np.arange(3, dtype=np.uint32), np.zeros(3, np.int32)
        nxt = np.empty(3, np.uint32)
        for row in (0, 1, 2):
            with pytest.raises(Gpt2qError, match="page table"):
                g._check(g._lib.gpt2q_page_out(g.h, 0, 5, arr, C.byref(t), row))
        with pytest.raises(Gpt2qError, match="page table"):
            g._check(g._lib.gpt2q_decode_paged(g.h, tok.ctypes.data, pos.ctypes.data, 3, arr, C.byref(t), None, nxt.ctypes.data))
        # a bad cache in the last layer: the earlier ones are not written either
        good = _ffi.PageTable(ids.data_ptr(), 3, 4, 4)
        arr[TINY.n_layer - 1].token_stride += 1
        with pytest.raises(Gpt2qError, match="16 bytes"):
            g._check(g._lib.gpt2q_page_out(g.h, 0, 5, arr, C.byref(good), 1))
        with pytest.raises(Gpt2qError, match="16 bytes"):
            g._check(g._lib.gpt2q_decode_paged(g.h, tok.ctypes.data, pos.ctypes.data, 3, arr, C.byref(good), None, nxt.ctypes.data))
        assert untouched(layers)


def test_expanded_outputs_are_refused_and_interleaved_ones_are_not():
    from smelt_b200.paged import Rotary

    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.empty(3, h, 64, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for h in (2, 2, 4))
    kv = PagedKV(*(torch.empty(8, 2, 16, 64, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2)))
    table = torch.arange(6, dtype=torch.int32, device="cuda").view(3, 2)
    pos = torch.tensor([17, 3, 30], dtype=torch.int32, device="cuda")
    rot = Rotary(64)
    for bad in (q[:1].expand(3, -1, -1), q[:, :1].expand(-1, 4, -1)):
        with pytest.raises(Gpt2qError, match="overlap"):
            kv.attend(q, table, pos, out=bad)
        with pytest.raises(Gpt2qError, match="overlap"):
            kv.append(k, v, table, pos, rotary=rot, q=q, q_out=bad)
    shared = PagedKV(*(x[:, :1].expand(-1, 2, -1, -1) for x in (kv.k, kv.v)))
    with pytest.raises(Gpt2qError, match="overlap"):
        shared.append(k, v, table, pos)
    want = kv.attend(q, table, pos)
    turned = kv.append(k, v, table, pos, rotary=rot, q=q)
    # rows every 192 elements, heads every 320: entries lie between one another and share nothing
    hold = torch.zeros(2 * 192 + 3 * 320 + 64, dtype=torch.bfloat16, device="cuda")
    woven = hold.as_strided((3, 4, 64), (192, 320, 1))
    assert torch.equal(kv.append(k, v, table, pos, rotary=rot, q=q, q_out=woven), turned)
    swapped = torch.zeros(4, 3, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    kv2 = PagedKV(kv.k.clone(), kv.v.clone())
    assert torch.equal(kv2.attend(q, table, pos, out=swapped), kv2.attend(q, table, pos, out=woven))
    assert want.shape == q.shape
