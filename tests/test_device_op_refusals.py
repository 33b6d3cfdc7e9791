"""Refused calls of the operators on device memory: every check is made on the host before anything is
launched, so these run without a GPU (the addresses below are never read)."""
import ctypes as C
import math

import pytest
import torch

from smelt_b200 import _ffi

A = 1 << 20  # a 16-byte aligned address


@pytest.fixture(scope="module")
def lib():
    from smelt_b200 import build
    build.build()
    return _ffi.load()


def cache(**kw):
    f = dict(k=A, v=A, dtype=1, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64, reserved=0,
             page_stride=2048, head_stride=1024, token_stride=64)
    f.update(kw)
    return _ffi.PagedKV(**f)


def table(**kw):
    f = dict(ids=A, n_rows=3, width=5, ld=5)
    f.update(kw)
    return _ffi.PageTable(**f)


def heads(**kw):
    f = dict(data=A, token_stride=128, head_stride=64)
    f.update(kw)
    return _ffi.Heads(**f)


def refused(lib, rc, text):
    assert rc == -1
    assert text in lib.gpt2q_last_error(None).decode(), lib.gpt2q_last_error(None)


def append(lib, kv=None, t=None, k=None, v=None, q=None, qo=None, dtype=1, nq=0, n=3, pos=A, seq=None, rot=None):
    r = [C.byref(x) if x is not None else None for x in (kv or cache(), t or table(), k or heads(), v or heads(), q, qo)]
    return lib.gpt2q_paged_append(*r, dtype, nq, n, pos, seq, None if rot is None else C.byref(rot), None, None)


def attend(lib, kv=None, t=None, lens=A, q=None, o=None, dtype=1, n=4, scale=0.1, window=0, work=A):
    r = [C.byref(x) for x in (kv or cache(), t or table())]
    return lib.gpt2q_paged_attention(*r, lens, C.byref(q or heads()), C.byref(o or heads()), dtype, n, scale, window, None,
                                     None, work, None)


CACHES = [
    (dict(k=None), "null cache"), (dict(v=None), "null cache"), (dict(dtype=3), "cache dtype"), (dict(dtype=-1), "cache dtype"),
    (dict(n_pages=0), "n_pages"), (dict(page_size=0), "page_size"), (dict(n_kv_heads=0), "n_kv_heads"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"),
    (dict(k=A + 8), "16 bytes"), (dict(v=A + 2), "16 bytes"), (dict(token_stride=68), "16 bytes"),
    (dict(head_stride=1), "16 bytes"), (dict(page_stride=2044), "16 bytes"), (dict(page_stride=-2048), "negative"),
    (dict(dtype=2), "dtype must be"), (dict(page_stride=1 << 36), "64 GB"),
]


@pytest.mark.parametrize("change,text", CACHES)
def test_caches(lib, change, text):
    refused(lib, append(lib, kv=cache(**change)), text)
    refused(lib, attend(lib, kv=cache(**change)), text)


@pytest.mark.parametrize("change", [dict(ids=None), dict(width=0), dict(ld=4), dict(n_rows=-1)])
def test_tables(lib, change):
    refused(lib, append(lib, t=table(**change)), "page table")
    refused(lib, attend(lib, t=table(**change)), "page table")


def test_append(lib):
    refused(lib, append(lib, n=-1), "n_tokens")
    refused(lib, append(lib, pos=None), "d_pos")
    refused(lib, append(lib, k=heads(data=None)), "null k or v")
    refused(lib, append(lib, v=heads(data=None)), "null k or v")
    refused(lib, append(lib, q=heads()), "come together")
    refused(lib, append(lib, qo=heads()), "come together")
    refused(lib, append(lib, q=heads(), qo=heads(), nq=0), "n_q_heads")
    refused(lib, append(lib, n=4), "more tokens than table rows")
    for dim in (0, 3, 66):
        refused(lib, append(lib, rot=_ffi.Rotary(dim=dim)), "rotary dim")
    refused(lib, append(lib, dtype=2), "dtype must be")
    assert append(lib, n=0) == 0


def test_rotary(lib):
    r = _ffi.Rotary()
    for dim, base in ((0, 10.0), (3, 10.0), (258, 10.0), (64, 0.0), (64, -1.0), (64, math.inf), (64, math.nan)):
        refused(lib, lib.gpt2q_rotary_init(C.byref(r), dim, 0, base), "rotary_init")
    refused(lib, lib.gpt2q_rotary_init(None, 64, 0, 10.0), "rotary_init")
    assert lib.gpt2q_rotary_init(C.byref(r), 64, 5, 10000.0) == 0
    assert r.dim == 64 and r.interleaved == 1
    for i in (0, 1, 31):
        assert abs(r.turns[i] * 2 * math.pi - 10000.0 ** (-2 * i / 64)) < 1e-15
    assert r.turns[32] == 0.0


def test_attention(lib):
    refused(lib, attend(lib, lens=None), "null")
    refused(lib, attend(lib, q=heads(data=None)), "null")
    refused(lib, attend(lib, o=heads(data=None)), "null")
    for n in (0, -2, 3):
        refused(lib, attend(lib, n=n), "n_heads")
    for s in (math.nan, math.inf):
        refused(lib, attend(lib, scale=s), "scale")
    refused(lib, attend(lib, window=-1), "window")
    refused(lib, attend(lib, work=None), "d_work")
    refused(lib, attend(lib, work=A + 4), "d_work")
    refused(lib, attend(lib, q=heads(data=A + 2)), "16 bytes")
    refused(lib, attend(lib, o=heads(token_stride=130)), "16 bytes")
    refused(lib, attend(lib, q=heads(head_stride=60)), "16 bytes")
    assert attend(lib, t=table(n_rows=0)) == 0
    assert lib.gpt2q_paged_attention_workspace(None, 4) == 0 and lib.gpt2q_paged_attention_workspace(C.byref(cache()), 0) == 0
    assert lib.gpt2q_paged_attention_workspace(C.byref(cache()), 4) >= 16


def logprobs(lib, x=A, dtype=0, ld=10, rows=2, vocab=10, temp=1.0, t=A, top=0, lp=A):
    return lib.gpt2q_logprobs(x, dtype, ld, rows, vocab, temp, t, 0, top, lp, None, None, None, None, None)


def grad(lib, x=A, dtype=0, ld=10, rows=2, vocab=10, temp=1.0, t=A, stats=A, lp=A, dx=2 * A, ldo=10):
    return lib.gpt2q_logprobs_grad(x, dtype, ld, rows, vocab, temp, t, 0, stats, lp, None, dx, ldo, None)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "null logits"), (dict(x=A + 2), "unaligned"), (dict(dtype=3), "dtype"), (dict(ld=9), "ld"),
    (dict(rows=-1), "n_rows"), (dict(vocab=0), "vocab"), (dict(temp=0.0), "temperature"), (dict(temp=-1.0), "temperature"),
    (dict(temp=math.nan), "temperature"), (dict(temp=math.inf), "temperature"), (dict(t=None), "targets")])
def test_logprobs_and_gradient(lib, change, text):
    refused(lib, logprobs(lib, **change), text)
    refused(lib, grad(lib, **change), text)


def test_logprobs_only(lib):
    for top in (-1, 11):
        refused(lib, logprobs(lib, top=top), "top")
    refused(lib, logprobs(lib, top=65, vocab=100, ld=100), "top")
    assert logprobs(lib, rows=0) == 0


def test_gradient_only(lib):
    refused(lib, grad(lib, stats=None), "null stats")
    refused(lib, grad(lib, dx=None), "null stats or dlogits")
    refused(lib, grad(lib, ldo=9), "ld_out")
    refused(lib, grad(lib, dx=2 * A + 1), "unaligned")
    refused(lib, grad(lib, dx=A, ldo=12), "in place")
    assert grad(lib, rows=0) == 0


def test_python_wrappers_refuse_host_tensors(lib):
    from smelt_b200.logprobs import token_logprobs, token_logprobs_grad
    from smelt_b200.paged import PagedKV, Rotary

    x = torch.zeros(2, 3, 4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        PagedKV(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 5))
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs_grad(torch.zeros(2, 5), None, None, None)
    with pytest.raises(ValueError, match="inv_freq"):
        Rotary(8, inv_freq=[1.0])
    with pytest.raises(_ffi.Gpt2qError):
        Rotary(7)


def test_tables_whose_rows_share_storage(lib):
    """The handle's page tables keep the tensor's stride, so that the call refuses rows that lie in one another."""
    from smelt_b200.gpu import _page_table

    t = torch.arange(8, dtype=torch.int32).view(2, 4)
    for x, ld in ((t, 4), (t[:, :3], 4), (t[:1], 4), (t[1:, 1:], 4), (torch.arange(4, dtype=torch.int32).expand(1, 4), 4)):
        p = _page_table(x)
        assert (p.ids, p.n_rows, p.width, p.ld) == (x.data_ptr(), *x.shape, ld)
    for x in (t[:1].expand(3, -1), t.view(-1).as_strided((3, 4), (2, 1))):
        p = _page_table(x)
        assert (p.n_rows, p.width, p.ld) == (3, 4, x.stride(0))
        p.ids = A  # never read
        refused(lib, append(lib, t=p), "page table")
        refused(lib, attend(lib, t=p), "page table")


def test_outputs_and_entries_that_overlap(lib):
    """An expanded or self-overlapping output, and for an append a cache whose entries share memory."""
    ok = dict(token_stride=256, head_stride=64)
    for bad in (dict(token_stride=0, head_stride=64), dict(token_stride=256, head_stride=0), dict(token_stride=64, head_stride=64),
                dict(token_stride=128, head_stride=64), dict(token_stride=56, head_stride=512), dict(token_stride=160, head_stride=320),
                dict(token_stride=-192, head_stride=64)):
        refused(lib, attend(lib, q=heads(**ok), o=heads(**bad)), "overlap")
        refused(lib, append(lib, q=heads(**ok), qo=heads(**bad), nq=4), "overlap")
    for bad in (dict(page_stride=0), dict(head_stride=0), dict(token_stride=0), dict(token_stride=32), dict(head_stride=512),
                dict(page_stride=1024)):
        refused(lib, append(lib, kv=cache(**bad)), "entries overlap")


def test_overlap_rule_against_every_element():
    """The rule, restated, against a count of every element: the library's is the same arithmetic."""
    import itertools
    import random

    def rule(n, a, m, b, dim):
        if n < 1 or m < 1:
            return False
        if a > b:
            a, b, n, m = b, a, m, n
        if (n > 1 and a < dim) or (m > 1 and b < dim):
            return True
        if n == 1 or m == 1 or b >= a * (n - 1) + dim:
            return False
        for j in range(1, m):
            i = j * b // a
            if (i < n and j * b - i * a < dim) or (i + 1 < n and (i + 1) * a - j * b < dim):
                return True
        return False

    rng = random.Random(1)
    seen = set()
    for _ in range(4000):
        n, m, dim = rng.randint(1, 6), rng.randint(1, 6), rng.randint(1, 5)
        a, b = rng.randint(0, 24), rng.randint(0, 24)
        at = [i * a + j * b + d for i, j, d in itertools.product(range(n), range(m), range(dim))]
        assert rule(n, a, m, b, dim) == (len(set(at)) < len(at)), (n, a, m, b, dim)
        seen.add(rule(n, a, m, b, dim))
    assert seen == {True, False}


def test_temperatures_too_small_to_divide_by(lib):
    for temp in (1e-45, 3e-39, 4.2e-39, 1e-36, 0.99e-30):
        refused(lib, logprobs(lib, temp=temp), "temperature")
        refused(lib, grad(lib, temp=temp), "temperature")
    assert logprobs(lib, rows=0, temp=1.01e-30) == 0 and grad(lib, rows=0, temp=1.01e-30) == 0


def test_a_copied_rotation_is_its_own(lib):
    """deepcopy (of a model that holds one) and pickling: the address is the copy's, not the original's."""
    import copy
    import pickle

    from smelt_b200.paged import Rotary

    r = Rotary(16, 1000.0, interleaved=True)
    turns = list(r.c.turns)
    for other in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert other.address == C.addressof(other.c) != r.address
        assert list(other.c.turns) == turns and (other.c.dim, other.c.interleaved) == (16, 1)
    assert r.address == C.addressof(r.c)
    assert copy.copy(r).address == r.address  # shares the structure, and keeps it


def test_pools_are_not_replaced(lib):
    from smelt_b200.paged import PagedKV

    kv = PagedKV.__new__(PagedKV)
    kv._pools = 1, 2
    assert (kv.k, kv.v) == (1, 2)
    for name in ("k", "v"):
        with pytest.raises(AttributeError):
            setattr(kv, name, 3)


def test_rows_longer_than_the_kernels_count(lib):
    """Ends of rows near 2^31 elements would pass 32 bits: (vector + 34) * 8 <= vocab was true for them."""
    for vocab in ((1 << 30) + 1, (1 << 31) - 1):
        refused(lib, logprobs(lib, vocab=vocab, ld=vocab), "2^30")
        refused(lib, grad(lib, vocab=vocab, ld=vocab, ldo=vocab), "2^30")
    assert logprobs(lib, rows=0, vocab=1 << 30, ld=1 << 30) == 0


def test_gradients_over_other_logits(lib):
    """dlogits in place are the logits themselves; one that starts elsewhere in them is refused, rows side by side are not."""
    for d in (4, -4, 36, 40, 76, -76, 48):  # rows of 10 floats, every 10 or 12
        refused(lib, grad(lib, dx=A + d, rows=3), "overlap")
    for d in (4, -4, 36, 44, 48, 52, -44, 96, 100):
        refused(lib, grad(lib, dx=A + d, rows=3, ld=12, ldo=12), "overlap")
    # accepted by the check: nothing of the kind is refused (without a GPU the launch fails, or nothing is launched)
    for d, ld in ((120, 10), (-120, 10), (40, 20), (-40, 20), (136, 12)):
        assert grad(lib, dx=A + d, rows=3, ld=ld, ldo=ld) != -1 if not torch.cuda.is_available() else True
