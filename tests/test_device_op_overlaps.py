"""Which outputs and caches the operators on device memory refuse because they share memory: on the host, without a GPU (the addresses
below are never read), against the bytes counted one by one. A call that passes the checks fails at its launch, as there is no GPU."""
import ctypes as C
import itertools
import random
import time

import pytest
import torch

from smelt_b200 import _ffi

A = 1 << 30
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are none")


@pytest.fixture(scope="module")
def lib():
    from smelt_b200 import build
    build.build()
    return _ffi.load()


def answer(lib, rc):
    """The message of a refusal, or None for a call that passed the checks."""
    assert rc != 0
    return lib.gpt2q_last_error(None).decode() if rc == -1 else None


def cache(k, v, pages, page, heads, dim, steps, dtype=1, scales=None):
    kv = _ffi.PagedKV(k=k, v=v, dtype=dtype, n_pages=pages, page_size=page, n_kv_heads=heads, head_dim=dim, reserved=int(scales is not None),
                      page_stride=steps[0], head_stride=steps[1], token_stride=steps[2])
    return kv if scales is None else _ffi.PagedKV8(kv, *scales)


FAR = cache(A << 8, A << 9, 2, 2, 2, 8, (32, 16, 8))


def heads(at, ts, hs):
    return _ffi.Heads(data=at, token_stride=ts, head_stride=hs)


def table(rows=1 << 20):
    return _ffi.PageTable(ids=A << 10, n_rows=rows, width=5, ld=5)


def append(lib, kv=FAR, n=3, k=None, v=None, q=None, o=None, nq=2, dtype=1, t=None):
    k, v = k or heads(A << 11, 32, 16), v or heads(A << 12, 32, 16)
    return answer(lib, lib.gpt2q_paged_append(C.byref(kv), C.byref(t or table()), C.byref(k), C.byref(v), q and C.byref(q), o and C.byref(o), dtype, nq if q else 0,
                                              n, A, None, None, None, None))


def read(lib, k, v, kv=FAR, n=3, dtype=1):
    return answer(lib, lib.gpt2q_paged_read(C.byref(kv), C.byref(table()), C.byref(k), C.byref(v), dtype, n, A, None, None, None))


def taken(at, n, m, ts, hs, dim, size):
    """The bytes of n x m runs, and whether two of the runs share one."""
    b = [at + (i * ts + j * hs) * size + e for i in range(n) for j in range(m) for e in range(dim * size)]
    return set(b), len(set(b)) < len(b)


def test_k_and_v_of_a_read(lib):
    rng = random.Random(1)
    dim, size = 8, 2
    seen = set()
    for _ in range(3000):
        n, m = rng.randint(1, 5), 2
        steps = [(rng.choice([8, 16, 24, 32, 40, 80]), rng.choice([8, 16, 24, 40, 64, 80])) for _ in range(2)]
        at = [A + 2 * rng.randint(0, 300) for _ in range(2)]
        (x, own_x), (y, own_y) = (taken(a, n, m, *s, dim, size) for a, s in zip(at, steps))
        got = read(lib, heads(at[0], *steps[0]), heads(at[1], *steps[1]), n=n)
        want = "entries of k or v overlap" if own_x or own_y else "k and v overlap" if x & y else None
        assert (want in got) if want else got is None, (at, n, steps, got, want)
        seen.add(want)
    assert len(seen) == 3


@pytest.mark.parametrize("dtype", [1, 8])
def test_a_cache_that_is_written(lib, dtype):
    """Strides of pages, heads and slots in any order, pools (and scales) beside, between and in one another."""
    rng = random.Random(2)
    dim, size = 16, 2 if dtype == 1 else 1
    kept = 0
    for _ in range(6000):
        n = [rng.randint(1, 3) for _ in range(3)]  # pages, heads, slots
        order, steps, at = rng.sample(range(3), 3), [0] * 3, 16
        for i in order:  # nested, or nearly
            steps[i] = at + 16 * rng.choice([0, 0, 0, 1, 2, -1])
            steps[i] = max(steps[i], 0)
            at = max(at, steps[i] * n[i])
        k = A + 16 * rng.randint(0, 30)
        v = A + 16 * rng.randint(0, 60)

        def bytes_of(base, st, run):
            b = [base + sum(x * s for x, s in zip(ix, st)) + e for ix in itertools.product(*map(range, n)) for e in range(run)]
            return set(b), len(set(b)) < len(b)
        sets = [bytes_of(x, [s * size for s in steps], dim * size) for x in (k, v)]
        scales = None
        if dtype == 8:
            ss = [rng.choice([1, 2, 3, 4, 6, 9]) for _ in range(3)]
            at = [A + 4 * rng.randint(200, 260), A + 4 * rng.randint(200, 800)]
            scales = (*at, ss[0], ss[1], ss[2])
            sets += [bytes_of(x, [s * 4 for s in ss], 4) for x in at]
        bad = any(own for _, own in sets) or any(x & y for (x, _), (y, _) in itertools.combinations(sets, 2))
        got = append(lib, cache(k, v, n[0], n[2], n[1], dim, steps, dtype, scales), n=1, k=heads(A << 11, 96, 32), v=heads(A << 12, 96, 32))
        assert ("entries overlap" in got) if bad else got is None, (n, steps, k - A, v - A, scales, got, bad)
        kept += not bad
    assert 300 < kept < 5700


def test_outputs_over_other_tensors(lib):
    """Queries, keys and values side by side, as a projection leaves them: in place, and not."""
    q, k, v = (heads(A + 16 * x, 48, 8) for x in (0, 2, 4))  # 2 + 2 + 2 heads of 8
    assert append(lib, k=k, v=v, q=q, o=q) is None
    for o in (k, v, heads(A + 16, 48, 8), heads(A + 96, 48, 8), heads(A, 48, 16), heads(A + 48, 48, 8)):
        assert "q_out" in append(lib, k=k, v=v, q=q, o=o)
    assert append(lib, n=1, k=k, v=v, q=q, o=heads(A, 999, 8)) is None  # one token has no stride
    assert append(lib, k=k, v=v, q=q, o=heads(A + 3 * 96, 16, 8)) is None
    assert "q_out overlaps the cache" in append(lib, cache(A, A << 9, 2, 2, 2, 8, (32, 16, 8)), q=heads(A << 13, 16, 8), o=heads(A + 32, 16, 8))
    # read: into the pools or the scales
    kv = cache(A, A + 4096, 4, 2, 2, 16, (64, 32, 16), 8, (A + 8192, A + 16384, 8, 2, 1))
    far = heads(A << 13, 32, 16)
    for at in (A, A + 4096 + 255, A + 8192 - 1, A + 16384 + 4 * 4):
        at = at // 2 * 2
        assert "overlaps the cache" in read(lib, heads(at, 32, 16), far, kv, n=1)
        assert "overlaps the cache" in read(lib, far, heads(at, 32, 16), kv, n=1)
    assert read(lib, heads(A + 256, 32, 16), far, kv, n=1) is None


def test_keys_and_values_in_one_pool(lib):
    """Taken where the same data go there twice."""
    kv, x = cache(A, A, 4, 2, 2, 16, (64, 32, 16)), heads(A << 13, 32, 16)
    assert append(lib, kv, k=x, v=x) is None
    assert "entries overlap" in append(lib, kv, k=x, v=heads(A << 14, 32, 16)) and "entries overlap" in append(lib, kv, k=x, v=heads(A << 13, 48, 16))
    assert "entries overlap" in append(lib, cache(A, A + 32, 4, 2, 2, 16, (64, 32, 16)), k=x, v=x)
    rot = _ffi.Rotary(dim=16)
    assert "entries overlap" in answer(lib, lib.gpt2q_paged_append(C.byref(kv), C.byref(table()), C.byref(x), C.byref(x), None, None, 1, 0, 3, A, None, C.byref(rot), None, None))
    assert "entries overlap" in answer(lib, lib.gpt2q_paged_commit(C.byref(kv), C.byref(table(5)), A << 11, A << 12, 3, 3, A << 13, None, None))
    for scales in ((A << 3, A << 3), (A << 3, A << 4)):
        kv8 = cache(A, A, 4, 2, 2, 16, (64, 32, 16), 8, (*scales, 8, 4, 2))
        assert append(lib, kv8, k=x, v=x) is None


def test_new_lengths_over_the_list_of_a_commit(lib):
    t = table(5)

    def commit(new, width=3, ld=7):
        return answer(lib, lib.gpt2q_paged_commit(C.byref(FAR), C.byref(t), A << 11, A, width, ld, new, None, None))
    for at in (A - 16, A, A + 8, A + 4 * 4 * 7 + 8):
        assert "d_accept" in commit(at)
    assert commit(A - 20) is None and commit(A + 4 * (4 * 7 + 3)) is None
    # five lengths lie between two rows of three of eight, and not of seven
    assert commit(A + 12, ld=8) is None and "d_accept" in commit(A + 12) and commit(A, width=0) is None
    t = table(2)
    assert commit(A + 12) is None


def test_checks_are_quick(lib):
    """A million pages, a hundred thousand tokens, heads outside and inside, pools that lie between one another."""
    for steps, off in (((1 << 15, 1 << 10, 1 << 7), 1 << 14), ((1 << 15, 1 << 7, 1 << 10), 1 << 14), ((1 << 10, 1 << 30, 1 << 7), 1 << 40)):
        kv = cache(A, A + 2 * off, 1 << 20, 8, 8, 128, steps)
        n = 100_000
        qkv = [heads((A << 11) + 2 * 128 * x, 24 * 128, 128) for x in (0, 8, 16)]
        t = time.perf_counter()
        for _ in range(100):
            assert append(lib, kv, n=n, k=qkv[1], v=qkv[2], q=qkv[0], o=qkv[0], nq=8) is None
        assert time.perf_counter() - t < 1.0  # 10 ms a call, of which the failing launch is most
