"""Paged key/value cache on the GPU (smelt_b200.paged) against a plain implementation in 64 bits.

Tolerances, derived before the first run. u = 2^-24 is half a step of fp32, e = eps/2 of the stored type.
 append: the angle is exact to 2^-24 turns times 2 pi and sincospif to 2 ulp, so sin and cos are within 2^-21;
   the two products and their sum add 3 u: |error| <= (|a| + |b|) 2^-20 + e |y| + the type's smallest step.
 attend: a score of D terms is within D u S, S = scale * sum |q_i k_i|, and exp's argument and exp itself add
   (|s| + 4) 2^-22; a weight's relative error counts twice (numerator and sum). Each of n keys adds one rounding to
   the sums: n u. Weights held in two 16-bit pieces add 2^-16 (bf16, the wider), and 2^-20 bounds three pieces for
   fp32 outputs. All times the largest |v|, plus e |o|."""
import math

import numpy as np
import pytest
import torch

from smelt_b200._ffi import Gpt2qError
from smelt_b200.paged import STATUS_PAGE, STATUS_POSITION, STATUS_ROW, PagedKV, Rotary

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY_STEP = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, kind="f32", scale=1.0):
    return torch.empty(shape, dtype=T[kind], device="cuda").normal_(0, scale, generator=g)


def pools(g, pages, heads, page, dim, kind, layout="hnd", fill=None):
    def one():
        shape = (pages, heads, page, dim) if layout == "hnd" else (pages, page, heads, dim)
        x = randn(g, *shape, kind=kind) if fill is None else torch.full(shape, fill, dtype=T[kind], device="cuda")
        return x if layout == "hnd" else x.transpose(1, 2)
    return one(), one()


def tables(rng, lens, page, pages):
    """Disjoint random pages of every row; entries past a row's last page are out of range."""
    need = [-(-n // page) for n in lens]
    assert sum(need) <= pages
    order = rng.permutation(pages)
    t = np.full((len(lens), max(1, max(need)) + 1), 1 << 30, np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(t).cuda()


def slots(table, row, pos, page):
    t = table.cpu().numpy()
    return [(int(t[r, p // page]), p % page) for r, p in zip(row, pos)]


def rotate64(x, pos, dim, interleaved, base):
    """(rotated, sum of magnitudes that entered each element) of x [tokens, heads, D] in 64 bits."""
    y = x.double().cpu().numpy().copy()
    mag = np.abs(y)
    i = np.arange(dim // 2)
    th = np.asarray(pos, np.float64)[:, None] * base ** (-2.0 * i / dim)
    c, s = np.cos(th)[:, None], np.sin(th)[:, None]
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)
    a, b = y[..., ia].copy(), y[..., ib].copy()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = np.abs(a) + np.abs(b)
    return y, mag


def close(got, want, tol, what=""):
    got = got.double().cpu().numpy()
    err = np.abs(got - want)
    over, worst = float(np.max(err - tol)), float(np.max(err))
    assert over <= 0, (what, over, worst)


APPEND = [  # io, cache, heads, kv, dim, rot, interleaved, page, layout
    ("bf16", "bf16", 8, 2, 128, 128, False, 16, "hnd"),
    ("f16", "f16", 6, 3, 64, 32, True, 7, "nhd"),
    ("f32", "f16", 0, 12, 64, 0, False, 64, "hnd"),
    ("f32", "f32", 5, 5, 80, 80, False, 1, "nhd"),
    ("f32", "bf16", 4, 1, 256, 64, True, 24, "hnd"),
    ("bf16", "bf16", 4, 2, 128, 64, False, 16, "hnd"),
    ("f32", "f16", 2, 2, 96, 32, False, 8, "nhd"),
    ("bf16", "bf16", 3, 1, 8, 6, False, 5, "hnd"),      # element by element: the dims are no multiples of 16
    ("f16", "f16", 2, 2, 24, 24, True, 3, "nhd"),
]


@pytest.mark.parametrize("io,cache,heads,kv,dim,rot,inter,page,layout", APPEND)
@pytest.mark.parametrize("counts,start", [([1], 0), ([1, 1, 1], 37), ([70, 1, 33], 5)])
def test_append_matches_definition(io, cache, heads, kv, dim, rot, inter, page, layout, counts, start):
    g, rng = gen(1), np.random.default_rng(2)
    lens = [n + start for n in counts]
    total = sum(-(-n // page) for n in lens)
    k_pool, v_pool = pools(g, total + 2, kv, page, dim, cache, layout)
    table = tables(rng, lens, page, total + 2)
    row = np.repeat(np.arange(len(counts)), counts)
    pos = np.concatenate([np.arange(n) + start for n in counts])
    # padding between the tokens: rows of position -1
    keep = np.sort(rng.permutation(len(pos) + 3)[: len(pos)])
    n = len(pos) + 3
    all_pos, all_row = np.full(n, -1, np.int32), np.zeros(n, np.int32)
    all_pos[keep], all_row[keep] = pos, row
    qkv = randn(g, n, heads + 2 * kv, dim, kind=io)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    before = [x.double().cpu().numpy() for x in (k_pool, v_pool)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rotary = Rotary(rot, 1000.0, interleaved=inter) if rot else None
    out = PagedKV(k_pool, v_pool).append(k, v, table, torch.from_numpy(all_pos).cuda(), seq=torch.from_numpy(all_row).cuda(),
                                         rotary=rotary, q=q if heads else None, status=status)
    assert int(status) == 0
    e = {t: torch.finfo(T[t]).eps / 2 for t in T}

    def turned(x):
        return rotate64(x, all_pos, rot, inter, 1000.0) if rot else (x.double().cpu().numpy(), np.abs(x.double().cpu().numpy()))
    want, mag = turned(k)
    tol = [np.zeros_like(b) for b in before]
    for i, (pg, o) in zip(keep, slots(table, row, pos, page)):
        before[0][pg, :, o], before[1][pg, :, o] = want[i], v[i].double().cpu().numpy()
        tol[0][pg, :, o] = (mag[i] * 2.0 ** -20 if rot else 0) + np.abs(want[i]) * e[cache] * 1.0001 + TINY_STEP[cache]
        tol[1][pg, :, o] = np.abs(before[1][pg, :, o]) * e[cache] + TINY_STEP[cache]
    close(k_pool, before[0], tol[0], "k")  # entries that no token names are unchanged
    close(v_pool, before[1], tol[1], "v")
    if heads:
        wq, mq = turned(q)
        raw = q.double().cpu().numpy()
        wq[all_pos < 0] = raw[all_pos < 0]
        close(out, wq, (mq * 2.0 ** -20 if rot else 0) + np.abs(wq) * e[io] * 1.0001 + TINY_STEP[io], "q")
        assert np.array_equal(out.double().cpu().numpy()[all_pos < 0], raw[all_pos < 0])


def test_append_far_positions_rows_by_index_and_queries_in_place():
    """Angles at positions past a million, each token its own row (no seq), q rotated where it lies."""
    g = gen(3)
    page, dim, n = 65536, 64, 4
    k_pool, v_pool = pools(g, 4, 1, page, dim, "f32")
    pos = [1_000_003, 0, 65_535, 1_048_575]
    table = torch.full((n, 16), -1, dtype=torch.int32, device="cuda")
    for i, p in enumerate(pos):
        table[i, p // page] = i
    k, v, q = randn(g, n, 1, dim), randn(g, n, 1, dim), randn(g, n, 3, dim)
    wk, mk = rotate64(k, pos, dim, False, 10000.0)
    wq, mq = rotate64(q, pos, dim, False, 10000.0)
    got = PagedKV(k_pool, v_pool).append(k, v, table, torch.tensor(pos, dtype=torch.int32, device="cuda"), rotary=Rotary(dim), q=q, q_out=q)
    assert got is q
    close(q, wq, mq * 2.0 ** -20 + np.abs(wq) * U)
    for i, p in enumerate(pos):
        close(k_pool[i, 0, p % page], wk[i, 0], mk[i, 0] * 2.0 ** -20 + np.abs(wk[i, 0]) * U)
        assert torch.equal(v_pool[i, 0, p % page], v[i, 0])


def test_append_own_frequencies_and_unaligned_inputs():
    """Frequencies given one by one; k, v and q start one element past a 16-byte boundary."""
    g = gen(4)
    n, dim = 5, 32
    k_pool, v_pool = pools(g, 5, 2, 4, dim, "bf16")
    flat = randn(g, n * 6 * dim + 1, kind="bf16")
    x = flat[1:].view(n, 6, dim)
    f = [0.5, 0.25, 3.0, 1e-3, 0.0, 1.0, 2.0, 7.0]
    pos = torch.tensor([0, 1, 2, 3, 9], dtype=torch.int32, device="cuda")
    table = torch.arange(5, dtype=torch.int32, device="cuda")[:, None].repeat(1, 3)
    q = PagedKV(k_pool, v_pool).append(x[:, 2:4], x[:, 4:], table, pos, rotary=Rotary(16, inv_freq=f), q=x[:, :2])
    y = x[:, :2].double().cpu().numpy()
    th = pos.cpu().numpy()[:, None] * np.array(f)
    a, b = y[..., :8].copy(), y[..., 8:16].copy()
    c, s = np.cos(th)[:, None], np.sin(th)[:, None]
    y[..., :8], y[..., 8:16] = a * c - b * s, b * c + a * s
    mag = np.abs(y)
    mag[..., :8] = mag[..., 8:16] = np.abs(a) + np.abs(b)
    close(q, y, mag * 2.0 ** -20 + np.abs(y) * (torch.finfo(torch.bfloat16).eps / 2) * 1.0001)  # half a step: 2^-8
    assert torch.equal(v_pool[4, :, 1], x[4, 4:])


def test_append_bad_pages_positions_and_rows_are_skipped():
    g = gen(5)
    k_pool, v_pool = pools(g, 3, 1, 4, 16, "f16")
    kv = PagedKV(k_pool, v_pool)
    before = k_pool.clone(), v_pool.clone()
    table = torch.tensor([[0, -1], [3, 1]], dtype=torch.int32, device="cuda")
    k, v = randn(g, 1, 1, 16, kind="f16"), randn(g, 1, 1, 16, kind="f16")
    for pos, row, bit in ((4, 0, STATUS_PAGE), (0, 1, STATUS_PAGE), (8, 0, STATUS_POSITION), (2 ** 31 - 1, 1, STATUS_POSITION),
                          (0, 2, STATUS_ROW), (0, -1, STATUS_ROW)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        kv.append(k, v, table, torch.tensor([pos], dtype=torch.int32, device="cuda"),
                  seq=torch.tensor([row], dtype=torch.int32, device="cuda"), status=status)
        assert int(status) == bit, (pos, row)
    assert torch.equal(k_pool, before[0]) and torch.equal(v_pool, before[1])


# ------------------------------------------------------------------------------------- attention
def attend64(q, k_pool, v_pool, table, lens, scale, window):
    """(out, lse, tolerance before the output's rounding) in 64 bits."""
    n, heads, dim = q.shape
    kv, page = k_pool.shape[1], k_pool.shape[2]
    group = heads // kv
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device="cuda")
    tol = torch.zeros(n, heads, 1, dtype=torch.float64, device="cuda")
    for r in range(n):
        ln = int(lens[r])
        if ln <= 0:
            continue
        lo = max(0, ln - window) if window else 0
        j = torch.arange(lo, ln, device="cuda")
        pages = table[r, torch.div(j, page, rounding_mode="floor")].long()
        K, V = k_pool[pages, :, j % page].double(), v_pool[pages, :, j % page].double()  # [keys, kv, dim]
        Q = q[r].double().view(kv, group, dim)
        s = torch.einsum("hgd,khd->hgk", Q, K) * scale
        S = torch.einsum("hgd,khd->hgk", Q.abs(), K.abs()) * scale
        w = torch.softmax(s, -1)
        out[r] = torch.einsum("hgk,khd->hgd", w, V).reshape(heads, dim)
        lse[r] = torch.logsumexp(s, -1).reshape(heads)
        rel = dim * U * S.amax(-1) + (s.abs().amax(-1) + 4) * 2.0 ** -22 + len(j) * U
        tol[r, :, 0] = (2 * rel * V.abs().amax((0, 2))[:, None]).reshape(heads)
    return out, lse, tol


def check_attend(q, k_pool, v_pool, table, lens, scale=None, window=0):
    n, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    lse = torch.empty(n, heads, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = PagedKV(k_pool, v_pool).attend(q, table, lens, scale=scale, window=window, lse=lse, status=status)
    want, wlse, tol = attend64(q, k_pool, v_pool, table, lens, scale, window)
    assert int(status) == 0
    e = torch.finfo(q.dtype).eps / 2
    pieces = 2.0 ** -20 if q.dtype == torch.float32 else 2.0 ** -16
    vmax = 8.0  # normal values; larger ones only widen the left side's bound
    t = tol + pieces * vmax + want.abs() * e * 1.01 + (2.0 ** -25 if q.dtype == torch.float16 else 0)
    t = torch.where((lens <= 0)[:, None, None], torch.zeros_like(t), t)
    close(out, want.cpu().numpy(), t.expand_as(want).cpu().numpy(), "out")
    fin = torch.isfinite(wlse)
    assert torch.equal(fin, torch.isfinite(lse)) and bool(torch.all(lse[~fin] == -math.inf))
    err = (lse.double() - wlse)[fin].abs()
    # the logarithm of the sum: its relative error (half of the bound above) and the rounding of the result
    lim = (tol[..., 0] / 2 + (wlse.abs() + 1) * 4 * U + 2.0 ** -20)[fin]
    assert bool(torch.all(err <= lim)), float((err - lim).max())
    return out


def attend_case(seed, lens, heads, kv, dim, io, cache, page, layout="hnd", window=0, scale=3.0):
    g, rng = gen(seed), np.random.default_rng(seed)
    total = sum(-(-max(0, n) // page) for n in lens) + 1
    k_pool, v_pool = pools(g, total, kv, page, dim, cache, layout)
    table = tables(rng, [max(0, n) for n in lens], page, total)
    # entries behind a row's last token, and pages nobody names, hold NaN
    used = torch.zeros(total, page, dtype=torch.bool, device="cuda")
    for r, n in enumerate(lens):
        j = torch.arange(max(0, n), device="cuda")
        used[table[r, torch.div(j, page, rounding_mode="floor")].long(), j % page] = True
    for p in (k_pool, v_pool):
        p.masked_fill_(~used[:, None, :, None], math.nan)
    q = randn(g, len(lens), heads, dim, kind=io, scale=scale)
    return check_attend(q, k_pool, v_pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window)


TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (8, 2), (7, 1), (16, 1), (40, 2), (15, 5)])
def test_attend_heads_and_types(io, cache, heads, kv):
    attend_case(7, [1, 33, 0, 200, 5, 16], heads, kv, 64, io, cache, 16)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 128, 136, 192, 256])
def test_attend_head_dims(io, cache, dim):
    attend_case(8, [1, 70, 31, -3, 129], 6, 2, dim, io, cache, 24, "nhd")


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("dim", [136, 160, 192, 80, 40])
def test_attend_after_a_call_full_of_nan(io, cache, dim):
    """What an earlier call left in shared memory does not reach the dims that a head does not fill."""
    g = gen(21)
    k_pool, v_pool = pools(g, 64, 8, 16, 256, cache, fill=math.nan)
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None].repeat(16, 1)
    out = PagedKV(k_pool, v_pool).attend(randn(g, 16, 16, 256, kind=io), table, torch.full((16,), 1024, dtype=torch.int32, device="cuda"))
    assert bool(torch.isnan(out).all())
    attend_case(22, [200, 17, 900] * 8, 8, 4, dim, io, cache, 16)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("page", [1, 3, 16, 64, 1000])
@pytest.mark.parametrize("window", [0, 1, 17, 250])
def test_attend_pages_and_windows(io, cache, page, window):
    attend_case(9, [15, 16, 17, 255, 1, 300], 4, 4, 64, io, cache, page, window=window)


@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("lens", [[9001], [1] * 700, [4097, 1, 0, 3000, 64], [0, 0, 0], [-1]])
def test_attend_long_and_many_rows(io, cache, lens):
    attend_case(10, lens, 4, 2, 128, io, cache, 16, scale=1.0)


@pytest.mark.parametrize("io,cache", TYPES)
def test_attend_one_key_returns_its_value(io, cache):
    g = gen(11)
    k_pool, v_pool = pools(g, 1, 2, 4, 64, cache)
    q = randn(g, 1, 6, 64, kind=io, scale=100.0)
    out = PagedKV(k_pool, v_pool).attend(q, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                                         torch.ones(1, dtype=torch.int32, device="cuda"))
    want = v_pool[0, :, 0].repeat_interleave(3, 0)[None].to(q.dtype)
    assert torch.equal(out, want)  # weight 1 / 1


@pytest.mark.parametrize("io,cache", TYPES)
def test_attend_extreme_values(io, cache):
    """Scores in the thousands on either side, a large query, and keys that are wholly alike."""
    g = gen(12)
    k_pool, v_pool = pools(g, 5, 1, 16, 64, cache)
    table = torch.arange(5, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([77], dtype=torch.int32, device="cuda")
    for scale in (300.0, 1e-4):
        check_attend(randn(g, 1, 4, 64, kind=io, scale=scale), k_pool, v_pool, table, lens)
    big = randn(g, 1, 4, 64, kind="f32", scale=1.0) * (1e6 if io == "f32" else 60000 / 4)
    check_attend(big.to(T[io]), k_pool, v_pool, table, lens, scale=1e-6)
    k_pool.fill_(0.5)
    check_attend(randn(g, 1, 4, 64, kind=io), k_pool, v_pool, table, lens)


def test_attend_infinite_key_gives_the_softmax_of_it():
    """A key of -inf score has weight 0; a row with NaN among its keys is NaN, its neighbour is not."""
    g = gen(13)
    k_pool, v_pool = pools(g, 4, 1, 8, 64, "f32")
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([10, 16], dtype=torch.int32, device="cuda")
    q = randn(g, 2, 1, 64).abs()
    k_pool[0, 0, 3] = -math.inf
    k_pool[2, 0, 1, 5] = math.nan
    out = PagedKV(k_pool, v_pool).attend(q, table, lens)
    keep = [i for i in range(10) if i != 3]
    K = torch.cat([k_pool[0, 0], k_pool[1, 0]])[keep].double()
    V = torch.cat([v_pool[0, 0], v_pool[1, 0]])[keep].double()
    want = torch.softmax(q[0, 0].double() @ K.T / 8, -1) @ V
    assert float((out[0, 0].double() - want).abs().max()) < 1e-5
    assert bool(torch.isnan(out[1]).all())


@pytest.mark.parametrize("io,cache", TYPES)
def test_attend_bad_pages_and_lengths_give_nan(io, cache):
    g = gen(14)
    k_pool, v_pool = pools(g, 6, 2, 16, 64, cache)
    table = torch.tensor([[0, 1, -1], [2, 6, 3], [4, 5, 0], [5, 7, 9]], dtype=torch.int32, device="cuda")
    q = randn(g, 4, 4, 64, kind=io)
    kv = PagedKV(k_pool, v_pool)

    def run(lens, window=0):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lse = torch.empty(4, 4, device="cuda")
        o = kv.attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), lse=lse, status=status, window=window)
        nan = torch.isnan(o).flatten(1)
        assert torch.equal(nan.all(1), nan.any(1)) and torch.equal(nan.all(1), torch.isnan(lse).all(1))
        return nan.all(1).tolist(), int(status)
    assert run([32, 16, 48, 0]) == ([False, False, False, False], 0)
    assert run([33, 17, 48, 16]) == ([True, True, False, False], STATUS_PAGE)
    assert run([32, 48, 49, 1]) == ([False, True, True, False], STATUS_PAGE | STATUS_POSITION)
    assert run([32, 48, 1000000, 1]) == ([False, True, True, False], STATUS_PAGE | STATUS_POSITION)
    assert run([32, 48, 2, 1], window=16) == ([False, False, False, False], 0)  # the bad page lies before the window


def test_attend_offsets_past_32_bits():
    """Pages whose entries start past 2^32 elements."""
    pages, page, dim = 1100, 32, 128
    stride = 1 << 22  # elements between pages: page 1025 starts past 2^32
    store = torch.empty(pages * stride, dtype=torch.float16, device="cuda")
    k_pool = store.as_strided((pages, 1, page, dim), (stride, page * dim, dim, 1))
    v_pool = store.as_strided((pages, 1, page, dim), (stride, page * dim, dim, 1), storage_offset=page * dim)
    g = gen(15)
    use = torch.tensor([[1025, 3, 1099, 1024]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    k, v = randn(g, 100, 1, dim, kind="f16"), randn(g, 100, 1, dim, kind="f16")
    kv = PagedKV(k_pool, v_pool)
    kv.append(k, v, use, torch.arange(100, dtype=torch.int32, device="cuda"), seq=torch.zeros(100, dtype=torch.int32, device="cuda"))
    assert torch.equal(k_pool[1099, 0, 5], k[69, 0]) and torch.equal(v_pool[1024, 0, 3], v[99, 0])
    check_attend(randn(g, 1, 4, dim, kind="f16"), k_pool, v_pool, use, lens)


def test_calls_without_tokens_or_rows():
    g = gen(19)
    k_pool, v_pool = pools(g, 2, 2, 16, 64, "bf16")
    kv = PagedKV(k_pool, v_pool)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    for table in (torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.empty(0, 3, dtype=torch.int32, device="cuda")):
        z = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
        assert kv.append(z, z, table, none, q=torch.empty(0, 8, 64, dtype=torch.bfloat16, device="cuda")).shape == (0, 8, 64)
    assert kv.attend(torch.empty(0, 8, 64, dtype=torch.bfloat16, device="cuda"), table, none).shape == (0, 8, 64)


def test_python_refusals_on_the_device():
    g = gen(20)
    k_pool, v_pool = pools(g, 2, 2, 16, 64, "bf16")
    kv = PagedKV(k_pool, v_pool)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    q = randn(g, 3, 8, 64, kind="bf16")
    k = randn(g, 3, 2, 64, kind="bf16")
    bad = [
        lambda: kv.attend(q.half(), table, lens),                       # neither the cache's type nor fp32
        lambda: kv.attend(q[:, :, :32], table, lens),
        lambda: kv.attend(q.transpose(0, 1).contiguous().transpose(0, 1)[:2], table, lens),
        lambda: kv.attend(q, table[:2], lens),
        lambda: kv.attend(q, table.long(), lens),
        lambda: kv.attend(q, table, lens.long()),
        lambda: kv.attend(q, table, lens.cpu()),
        lambda: kv.attend(q, table, lens, out=q.float()),
        lambda: kv.attend(q, table, lens, lse=torch.empty(3, 8, dtype=torch.float64, device="cuda")),
        lambda: kv.append(k, k[:2], table, lens),
        lambda: kv.append(k, k, table, lens[:2]),
        lambda: kv.append(k, k, table, lens, q_out=q),
        lambda: kv.append(k, k, table, lens, status=lens),
        lambda: PagedKV(k_pool, v_pool.float()),
        lambda: PagedKV(k_pool, v_pool.transpose(1, 2).contiguous().transpose(1, 2)),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(Gpt2qError, match="n_heads"):
        kv.attend(q[:, :7], table, lens)
    with pytest.raises(Gpt2qError, match="window"):
        kv.attend(q, table, lens, window=-1)
    with pytest.raises(Gpt2qError, match="16 bytes"):
        kv.attend(torch.zeros(3 * 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 8, 64), table, lens)
    assert kv.attend(q, table, lens).shape == q.shape


def test_attend_strided_inputs_outputs_and_table():
    g = gen(16)
    k_pool, v_pool = pools(g, 8, 2, 16, 64, "bf16")
    wide = torch.arange(8, dtype=torch.int32, device="cuda").repeat(3, 2)[:, 1:7]
    lens = torch.tensor([60, 3, 96], dtype=torch.int32, device="cuda")
    qkv = randn(g, 3, 12, 64, kind="bf16")
    q = qkv[:, 4:8]
    hold = torch.full((3, 9, 72), 7.0, dtype=torch.bfloat16, device="cuda")
    out = hold[:, 2:6, :64]
    kv = PagedKV(k_pool, v_pool)
    kv.attend(q, wide, lens, out=out)
    assert torch.equal(out, kv.attend(q.contiguous(), wide.contiguous(), lens))
    mask = torch.ones_like(hold, dtype=torch.bool)
    mask[:, 2:6, :64] = False
    assert bool((hold[mask] == 7.0).all())


def test_attend_is_deterministic_captured_and_replayed_on_another_stream():
    g = gen(17)
    lens = torch.tensor([900, 64, 2100], dtype=torch.int32, device="cuda")
    k_pool, v_pool = pools(g, 200, 2, 16, 128, "bf16")
    table = torch.arange(3 * 140, dtype=torch.int32, device="cuda").view(3, 140) % 200
    q = randn(g, 3, 8, 128, kind="bf16")
    kv = PagedKV(k_pool, v_pool)
    first = kv.attend(q, table, lens)
    for _ in range(3):
        assert torch.equal(kv.attend(q, table, lens), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):  # two graphs, each with its own workspace
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                out = kv.attend(q, table, lens)
            graphs.append((gr, out))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    q2 = randn(g, 3, 8, 128, kind="bf16")
    for new_lens in ([1, 0, 700], [2200, 2201, 2240]):
        lens.copy_(torch.tensor(new_lens, dtype=torch.int32))
        q.copy_(q2)
        want = kv.attend(q, table, lens)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want)


def test_tokens_appended_one_by_one_are_attended():
    """Three sequences grow token by token from ragged prompts; each step's output matches dense attention
    over everything appended so far."""
    g = gen(18)
    kvh, heads, dim, page, steps = 2, 6, 64, 8, 12
    prompts = [5, 1, 19]
    n = len(prompts)
    k_pool, v_pool = pools(g, 20, kvh, page, dim, "f32", fill=math.nan)
    kv = PagedKV(k_pool, v_pool)
    table = tables(np.random.default_rng(0), [p + steps for p in prompts], page, 20)
    rot = Rotary(dim)
    ks, vs = [[] for _ in prompts], [[] for _ in prompts]

    def take(k, pos, row, v):
        wk, _ = rotate64(k, pos, dim, False, 10000.0)
        for i, r in enumerate(row):
            ks[r].append(wk[i])
            vs[r].append(v[i].double().cpu().numpy())
    tokens = sum(prompts)
    row = np.repeat(np.arange(n), prompts)
    pos = np.concatenate([np.arange(p) for p in prompts])
    k, v = randn(g, tokens, kvh, dim), randn(g, tokens, kvh, dim)
    kv.append(k, v, table, torch.tensor(pos, dtype=torch.int32, device="cuda"), seq=torch.tensor(row, dtype=torch.int32, device="cuda"), rotary=rot)
    take(k, pos, row, v)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    for _ in range(steps):
        k, v, q = randn(g, n, kvh, dim), randn(g, n, kvh, dim), randn(g, n, heads, dim)
        at = lens.clone()
        turned = kv.append(k, v, table, at, rotary=rot, q=q)
        take(k, at.cpu().numpy(), range(n), v)
        lens += 1
        out = kv.attend(turned, table, lens)
        wq, _ = rotate64(q, at.cpu().numpy(), dim, False, 10000.0)
        for r in range(n):
            K, V = np.stack(ks[r]), np.stack(vs[r])  # [keys, kv, dim]
            for h in range(heads):
                s = K[:, h // 3] @ wq[r, h] / 8
                w = np.exp(s - s.max())
                o = (w / w.sum()) @ V[:, h // 3]
                # scores of O(10): rotation 2^-20 and accumulation, as above, leave about 1e-5 of |v| < 5
                assert np.abs(out[r, h].double().cpu().numpy() - o).max() < 5e-5
