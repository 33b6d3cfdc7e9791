"""Refused calls of the 8-bit cache and of drafted tokens' operators: checks on the host, without a GPU (the addresses below are
never read)."""
import ctypes as C
import math

import pytest

from smelt_b200 import _ffi

A = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from smelt_b200 import build
    build.build()
    return _ffi.load()


def cache(k_scale=A, v_scale=A, sps=32, shs=16, sts=1, **kw):
    f = dict(k=A, v=A, dtype=8, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, reserved=1,
             page_stride=2048, head_stride=1024, token_stride=64)
    f.update(kw)
    return _ffi.PagedKV8(_ffi.PagedKV(**f), k_scale, v_scale, sps, shs, sts)


def table(**kw):
    return _ffi.PageTable(**(dict(ids=A, n_rows=3, width=5, ld=5) | kw))


def heads(**kw):
    return _ffi.Heads(**(dict(data=A, token_stride=128, head_stride=64) | kw))


def ref(x):
    return None if x is None else C.byref(x)


def append(lib, kv=None, t=None, k=None, v=None, dtype=1, n=3, pos=A, slot=None):
    return lib.gpt2q_paged_append_at(ref(kv or cache()), ref(t or table()), ref(k or heads()), ref(v or heads()), None, None, dtype, 0, n, pos,
                                     slot, None, None, None, None)


def read(lib, kv=None, t=None, k=None, v=None, dtype=1, n=3, pos=A, seq=None):
    return lib.gpt2q_paged_read(ref(kv or cache()), ref(t or table()), ref(k or heads()), ref(v or heads()), dtype, n, pos, seq, None, None)


def attend(lib, kv=None, dtype=1):
    return lib.gpt2q_paged_attention(ref(kv or cache()), ref(table()), A, ref(heads()), ref(heads()), dtype, 4, 0.1, 0, None, None, A, None)


def tree(lib, kv=None, t=None, lens=A, first=A, mask=None, words=0, q=None, o=None, dtype=1, heads_n=2, n=5, scale=0.1, work=A):
    return lib.gpt2q_paged_tree_attention(ref(kv or cache()), ref(t or table()), lens, first, mask, words, ref(q or heads()), ref(o or heads()),
                                          dtype, heads_n, n, scale, None, None, work, None)


def commit(lib, kv=None, t=None, lens=A, accept=2 * A, width=3, ld=3, new=3 * A):
    return lib.gpt2q_paged_commit(ref(kv or cache()), ref(t or table()), lens, accept, width, ld, new, None, None)


def refused(lib, rc, text):
    assert rc == -1
    assert text in lib.gpt2q_last_error(None).decode(), lib.gpt2q_last_error(None)


@pytest.mark.parametrize("change,text", [
    (dict(reserved=0), "GPT2Q_SCALED"), (dict(k_scale=None), "null scales"), (dict(v_scale=None), "null scales"), (dict(k_scale=A + 2), "unaligned scales"),
    (dict(sps=-1), "scale stride"), (dict(shs=1 << 40), "scale stride"), (dict(head_dim=72, token_stride=80, head_stride=1280, page_stride=2560), "multiple of 16"),
    (dict(dtype=7), "cache dtype"), (dict(dtype=10), "cache dtype"), (dict(dtype=3), "cache dtype"), (dict(k=A + 8), "16 bytes"),
    (dict(token_stride=72), "16 bytes"), (dict(head_dim=272), "head_dim"), (dict(n_pages=0), "n_pages")])
def test_caches(lib, change, text):
    for call in (append, read, attend, tree, commit):
        refused(lib, call(lib, kv=cache(**change)), text)


@pytest.mark.parametrize("code", [8, 9])
def test_types(lib, code):
    for dtype in (3, 8, 9, -1):
        for call in (append, read, attend, tree):
            refused(lib, call(lib, kv=cache(dtype=code), dtype=dtype), "dtype must be")


def test_entries_or_scales_that_share_memory(lib):
    for change in (dict(sts=0), dict(shs=0), dict(sps=0), dict(token_stride=48), dict(head_stride=16)):
        refused(lib, append(lib, kv=cache(**change)), "overlap")
        refused(lib, commit(lib, kv=cache(**change)), "overlap")
    refused(lib, read(lib, k=heads(token_stride=64)), "overlap")
    refused(lib, read(lib, v=heads(head_stride=32)), "overlap")
    refused(lib, tree(lib, o=heads(head_stride=0)), "overlap")


def test_append_and_read(lib):
    for call in (append, read):
        refused(lib, call(lib, n=-1), "n_tokens")
        refused(lib, call(lib, pos=None), "d_pos")
        refused(lib, call(lib, k=heads(data=None)), "null k or v")
        refused(lib, call(lib, v=heads(data=None)), "null k or v")
        refused(lib, call(lib, n=4), "more tokens than table rows")
        refused(lib, call(lib, t=table(ld=4)), "page table")
        assert call(lib, n=0) == 0
    refused(lib, read(lib, k=heads(data=A + 1)), "unaligned k or v")


def test_tree(lib):
    refused(lib, tree(lib, lens=None), "null")
    refused(lib, tree(lib, first=None), "null d_first")
    refused(lib, tree(lib, mask=A, words=0), "mask_words")
    refused(lib, tree(lib, n=-1), "n_tokens")
    refused(lib, tree(lib, n=1 << 30), "too many tokens")
    for n in (0, 3, -2):
        refused(lib, tree(lib, heads_n=n), "n_heads")
    for s in (math.nan, math.inf):
        refused(lib, tree(lib, scale=s), "scale")
    refused(lib, tree(lib, work=None), "d_work")
    refused(lib, tree(lib, work=A + 8), "d_work")
    refused(lib, tree(lib, q=heads(data=A + 2)), "16 bytes")
    refused(lib, tree(lib, o=heads(data=None)), "null")
    assert tree(lib, n=0, first=None) == 0 and tree(lib, t=table(n_rows=0)) == 0
    size = lib.gpt2q_paged_tree_attention_workspace
    assert size(None, 4, 4) == 0 and size(ref(cache()), 0, 4) == 0 and size(ref(cache()), 4, -1) == 0 and size(ref(cache()), 4, 5) >= 16


def test_commit(lib):
    refused(lib, commit(lib, lens=None), "null")
    refused(lib, commit(lib, accept=None), "null")
    refused(lib, commit(lib, new=None), "null")
    refused(lib, commit(lib, width=-1), "width")
    refused(lib, commit(lib, ld=2), "ld < width")
    for at in (A, A + 8, A - 8):  # 3 rows
        refused(lib, commit(lib, new=at), "d_new_lens")
    assert commit(lib, t=table(n_rows=0)) == 0
