"""The 8-bit paged cache on the GPU: codes and scales against the same fp32 operations and against 64 bits, reading back, and
attention of one new token (paged_oracle.py derives the bounds).

A rotated key is within (|a| + |b|) 2^-20 of the exact one before it is quantised (angle, sine and cosine, products); its code is then
off by half a step of the codes: scale / 2 (int8); e4m3 2^-4 of the value, at least scale * 2^-10 (half a step of its smallest
numbers). The scale itself and the product with its inverse are fp32 operations: 4 u relative."""
import math

import numpy as np
import pytest
import torch

from smelt_b200._ffi import Gpt2qError
from smelt_b200.paged import STATUS_PAGE, STATUS_POSITION, STATUS_ROW, PagedKV, Rotary

from .paged_oracle import T, TOP, U, Cache, attention64, bound_of, close, gen, quantise, randn, tables

pytestmark = pytest.mark.gpu
CODES = ["i8", "e4m3"]
IO = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def rotate64(x, pos, dim, interleaved, base):
    y = x.double().clone()
    mag = y.abs()
    i = torch.arange(dim // 2, device="cuda")
    th = pos.double()[:, None] * base ** (-2.0 * i.double() / dim)
    c, s = torch.cos(th)[:, None], torch.sin(th)[:, None]
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def bits(x):
    return x.view(torch.int8)


STORE = [  # io, kv heads, dim, page, layout
    ("f32", 12, 64, 64, "hnd"), ("bf16", 8, 128, 16, "nhd"), ("f16", 2, 80, 7, "hnd"), ("f32", 1, 256, 1, "nhd"),
    ("bf16", 3, 16, 5, "hnd"), ("f16", 25, 144, 24, "nhd"),
]


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("io,kv,dim,page,layout", STORE)
@pytest.mark.parametrize("counts,start,aligned", [([1], 0, True), ([70, 1, 33], 5, True), ([3, 9], 2, False)])
def test_codes_are_those_of_the_fp32_operations(kind, io, kv, dim, page, layout, counts, start, aligned):
    g, rng = gen(1), np.random.default_rng(2)
    lens = [n + start for n in counts]
    pages = sum(-(-n // page) for n in lens) + 1
    c = Cache(g, pages, kv, page, dim, kind, layout)
    table = tables(rng, lens, page, pages)
    row = i32(np.repeat(np.arange(len(counts)), counts))
    pos = i32(np.concatenate([np.arange(n) + start for n in counts]))
    n = len(pos)
    hold = randn(g, n, 2 * kv, dim + (0 if aligned else 1), kind=io, scale=2.0)[..., :dim]
    k, v = hold[:, :kv], hold[:, kv:]
    k[0, 0] = 0.0                      # an entry of zeros
    v[n - 1, kv - 1, 1:] = 0.0         # one element of a size
    if n > 2:
        k[1, 0] *= 2.0 ** -8
    before = [p.clone() for p in c.pools], [s.clone() for s in c.scales]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.kv.append(k, v, table, pos, seq=row, status=status)
    assert int(status) == 0
    at = table[row.long(), (pos // page).long()].long(), (pos % page).long()
    for i, x in enumerate((k, v)):
        code, scale = quantise(x, kind)
        bits(before[0][i])[at[0], :, at[1]] = bits(code)
        before[1][i][at[0], :, at[1]] = scale
        assert torch.equal(bits(c.pools[i]), bits(before[0][i])) and torch.equal(c.scales[i], before[1][i])
    # read back, in every type: one rounding of the value; rows of padding between them
    keep = torch.arange(n, device="cuda") % 3 != 1
    for to in IO:
        got = c.kv.read(table, torch.where(keep, pos, -1), seq=row, dtype=T[to])
        for x, y in zip(got, c.values):
            want = y[at[0], :, at[1]]
            f = (want.float()).to(T[to])  # code * scale rounded to fp32, then to the type
            assert x.dtype == T[to] and torch.equal(x, torch.where(keep[:, None, None], f, 0.0))


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("io,heads,kv,dim,rot,inter,aligned", [
    ("bf16", 8, 2, 128, 128, False, True), ("f16", 6, 3, 64, 32, True, True), ("f32", 4, 1, 256, 64, True, True), ("f32", 5, 5, 80, 80, False, True),
    ("bf16", 3, 1, 16, 6, False, True), ("f16", 2, 2, 48, 40, True, True), ("f32", 4, 2, 128, 128, False, False), ("bf16", 2, 2, 64, 64, True, False)])
def test_rotated_keys(kind, io, heads, kv, dim, rot, inter, aligned):
    g, rng = gen(3), np.random.default_rng(4)
    page, lens = 8, [40, 17]
    c = Cache(g, 9, kv, page, dim, kind)
    table = tables(rng, lens, page, 9)
    row = i32([0] * 30 + [1] * 9 + [0, 0])
    pos = i32(list(range(10, 40)) + list(range(8, 17)) + [-1, -1])
    n = len(pos)
    qkv = randn(g, n, heads + 2 * kv, dim + (0 if aligned else 1), kind=io)[..., :dim]
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    turned = c.kv.append(k, v, table, pos, seq=row, rotary=Rotary(rot, 1000.0, interleaved=inter), q=q)
    real = pos >= 0
    wk, mk = rotate64(k, pos.clamp(min=0), rot, inter, 1000.0)
    wq, mq = rotate64(q, pos.clamp(min=0), rot, inter, 1000.0)
    e = torch.finfo(T[io]).eps / 2
    close(turned[real], wq[real], (mq * 2.0 ** -20 + wq.abs() * e * 1.0001 + (2.0 ** -24 if io == "f16" else 0))[real])
    assert torch.equal(turned[~real], q[~real])
    at = table[row.long(), (pos.clamp(min=0) // page).long()].long()[real], (pos % page).long()[real]
    got = c.values[0][at[0], :, at[1]]
    want, mag = wk[real], mk[real]
    scale = want.abs().amax(-1, keepdim=True) / TOP[kind]
    err = (mag.amax(-1, keepdim=True) * 2.0 ** -20).expand_as(want)
    step = scale / 2 if kind == "i8" else torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    close(got, want, step * (1 + 2.0 ** -10) + 2 * err + want.abs() * 8 * U)
    # in place, and from slots that are not the positions
    slot = torch.where(real, torch.where(row == 0, pos - 10, pos - 8), -5)
    c2 = Cache(gen(3), 9, kv, page, dim, kind)
    mine = q.clone()
    out = c2.kv.append(k, v, table, pos, seq=row, rotary=Rotary(rot, 1000.0, interleaved=inter), q=mine, q_out=mine, slot=slot)
    assert out is mine and torch.equal(mine, turned)
    for i in range(2):
        a = c2.pools[i][table[row.long(), (slot.clamp(min=0) // page).long()].long()[real], :, (slot % page).long()[real]]
        assert torch.equal(bits(a), bits(c.pools[i][at[0], :, at[1]].contiguous()))


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("aligned", [True, False])
def test_entries_that_have_no_scale(kind, aligned):
    """Zeros, numbers under 2^-100, the largest fp32 numbers, infinities and NaN."""
    c = Cache(gen(5), 1, 1, 8, 32, kind)
    x = torch.zeros(6, 1, 32 + (not aligned), device="cuda")[..., :32]
    x[1] = 2.0 ** -101
    x[2] = 2.0 ** -100
    x[3, 0, :2] = torch.tensor([3.4028234e38, -1e38])
    x[4, 0, 7], x[4, 0, 8] = math.inf, 1.0
    x[5, 0, 31] = math.nan
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    seq = torch.zeros(6, dtype=torch.int32, device="cuda")
    c.kv.append(x, x, table, torch.arange(6, dtype=torch.int32, device="cuda"), seq=seq)
    for s, p in zip(c.scales, c.pools):
        assert s[0, 0, :2].tolist() == [0.0, 0.0] and bool(torch.isnan(s[0, 0, 4:6]).all())
        assert bool((bits(p)[0, 0, [0, 1, 4, 5]] == 0).all())
    k, v = c.kv.read(table, torch.arange(6, dtype=torch.int32, device="cuda"), seq=seq, dtype=torch.float32)
    for y in (k, v):
        assert bool((y[:2] == 0).all()) and bool(torch.isnan(y[4:]).all())
        assert torch.equal(y[2], torch.full_like(y[2], 2.0 ** -100)) or bool(((y[2] - 2.0 ** -100).abs() <= 2.0 ** -122).all())
        assert bool(((y[3] - x[3]).abs() <= 3.4028234e38 / (254 if kind == "i8" else 16)).all())


def test_bad_pages_positions_and_rows():
    for kind in CODES:
        c = Cache(gen(5), 3, 1, 4, 16, kind)
        before = [bits(x).clone() for x in c.pools]
        table = i32([[0, -1], [3, 1]])
        k = randn(gen(6), 1, 1, 16, kind="f16")
        for pos, slot, row, bit in ((4, None, 0, STATUS_PAGE), (0, None, 1, STATUS_PAGE), (8, None, 0, STATUS_POSITION), (2 ** 31 - 1, None, 1, STATUS_POSITION),
                                    (0, None, 2, STATUS_ROW), (0, None, -1, STATUS_ROW), (0, -1, 0, STATUS_POSITION), (0, 8, 0, STATUS_POSITION),
                                    (900, 4, 0, STATUS_PAGE)):
            for kk in (k, torch.zeros(17, dtype=torch.float16, device="cuda")[1:].view(1, 1, 16)):
                status = torch.zeros(1, dtype=torch.int32, device="cuda")
                c.kv.append(kk, kk, table, i32([pos]), seq=i32([row]), status=status, slot=None if slot is None else i32([slot]))
                assert int(status) == bit, (pos, slot, row)
            if slot is None:
                status = torch.zeros(1, dtype=torch.int32, device="cuda")
                x, y = c.kv.read(table, i32([pos]), seq=i32([row]), status=status)
                assert int(status) == bit and bool(torch.isnan(x).all()) and bool(torch.isnan(y).all())
        assert all(torch.equal(bits(a), b) for a, b in zip(c.pools, before))


@pytest.mark.parametrize("cache,io", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("dim,layout", [(8, "hnd"), (128, "nhd"), (200, "hnd")])
def test_read_of_float_caches(cache, io, dim, layout):
    g, rng = gen(7), np.random.default_rng(8)
    lens, page = [301, 1, 45], 16
    c = Cache(g, 25, 3, page, dim, cache, layout)
    table = tables(rng, lens, page, 25)
    row = i32(np.repeat(np.arange(3), lens))
    pos = i32(np.concatenate([np.arange(n) for n in lens]))
    mix = torch.randperm(len(pos), generator=g, device="cuda")
    row, pos = row[mix], pos[mix]
    n = len(pos)
    want = [p[table[row.long(), (pos // page).long()].long(), :, (pos % page).long()].to(T[io]) for p in c.pools]
    got = c.kv.read(table, pos, seq=row, dtype=T[io])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # into strided tensors of the caller's, aligned and not; what lies between is left as it was
    for odd in (0, 1):
        hold = torch.full((n, 7, dim + 8 + odd), 3.0, dtype=T[io], device="cuda")
        k, v = hold[:, :3, :dim], hold[:, 4:, odd:dim + odd]
        r = c.kv.read(table, pos, seq=row, k=k, v=v)
        assert r[0] is k and r[1] is v and torch.equal(k, want[0]) and torch.equal(v, want[1])
        hold[:, :3, :dim], hold[:, 4:, odd:dim + odd] = 3.0, 3.0
        assert bool((hold == 3.0).all())


# ------------------------------------------------------------------------------------- attention of one new token
def attend_case(seed, lens, heads, kv, dim, io, cache, page, layout="hnd", window=0, scale=3.0, sizes=0.5, spoil=True):
    g, rng = gen(seed), np.random.default_rng(seed)
    there = [max(0, n) for n in lens]
    pages = sum(-(-n // page) for n in there) + 1
    c = Cache(g, pages, kv, page, dim, cache, layout, sizes)
    table = tables(rng, there, page, pages)
    values = c.values
    if spoil:
        c.spoil(c.used(table, there))
    q = randn(g, len(lens), heads, dim, kind=io, scale=scale)
    n, lse = len(lens), torch.empty(len(lens), heads, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = c.kv.attend(q, table, i32(lens), window=window, lse=lse, status=status)
    assert int(status) == 0 and out.dtype == T[io]
    for r in range(n):
        ln = there[r]
        if ln == 0:
            assert bool((out[r] == 0).all()) and bool((lse[r] == -math.inf).all())
            continue
        keys = torch.arange(max(0, ln - window) if window else 0, ln, device="cuda")
        want, wl, tol, size, rel, vmax = attention64(q[r:r + 1], values, table[r], keys, torch.ones(1, len(keys), dtype=torch.bool, device="cuda"), dim ** -0.5)
        close(out[r:r + 1], want, bound_of(tol, size, vmax, want, io, cache), ("out", r))
        close(lse[r:r + 1], wl, rel + (wl.abs() + 1) * 4 * U + 2.0 ** -20, ("lse", r))
    return out


@pytest.mark.parametrize("cache", CODES)
@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("heads,kv", [(1, 1), (12, 12), (8, 2), (7, 1), (16, 1), (40, 2), (15, 5)])
def test_attend_heads_and_types(cache, io, heads, kv):
    attend_case(7, [1, 33, 0, 200, 5, 16], heads, kv, 64, io, cache, 16)


@pytest.mark.parametrize("cache", CODES)
@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 128, 144, 192, 256])
@pytest.mark.parametrize("page", [24, 32])
def test_attend_head_dims(cache, io, dim, page):
    attend_case(8, [1, 70, 31, -3, 129], 6, 2, dim, io, cache, page, "nhd")


@pytest.mark.parametrize("cache", CODES)
@pytest.mark.parametrize("page", [1, 3, 16, 64, 1000])
@pytest.mark.parametrize("window", [0, 1, 17, 250])
def test_attend_pages_and_windows(cache, page, window):
    for io in IO:
        attend_case(9, [15, 16, 17, 255, 1, 300], 4, 4, 64, io, cache, page, window=window)


@pytest.mark.parametrize("cache", CODES)
@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("lens", [[9001], [1] * 700, [4097, 1, 0, 3000, 64], [0, 0, 0], [-1]])
def test_attend_long_and_many_rows(cache, io, lens):
    attend_case(10, lens, 4, 2, 128, io, cache, 16, scale=1.0)


@pytest.mark.parametrize("cache", CODES)
@pytest.mark.parametrize("lens", [[0, 5, 0, 0, 40] * 110 + [3000, 0, 1, 2500] + [2] * 40, [2100, 1], [0, 17, 0] * 171 + [600]])
def test_attend_short_rows_between_empty_and_long_ones(cache, lens):
    """More rows than threads, ranges that begin before a row's first key or end there, long rows at the list's end."""
    attend_case(13, lens, 6, 3, 64, "bf16", cache, 16, scale=1.0)


@pytest.mark.parametrize("cache", CODES)
@pytest.mark.parametrize("io", IO)
def test_attend_scales_of_very_different_sizes(cache, io):
    """Entries' sizes over ten powers of ten: the bound is in units of the largest value, whatever comes first."""
    attend_case(11, [700, 64, 33], 8, 2, 64, io, cache, 16, scale=1e-3, sizes=4.0)


@pytest.mark.parametrize("cache", CODES)
def test_attend_queries_out_of_the_range_of_fp16(cache):
    g = gen(12)
    c = Cache(g, 3, 1, 16, 64, cache)
    table = i32([[2, 0, 1]])
    base = randn(g, 1, 4, 64)
    for io in ("f32", "bf16"):
        for f in (2.0 ** 100, 2.0 ** -100, 2.0 ** 20):
            q = (base * f).to(T[io])
            out = c.kv.attend(q, table, i32([41]), scale=1 / (8 * f))
            want, _, tol, size, _, vmax = attention64(q, c.values, table[0], torch.arange(41, device="cuda"), torch.ones(1, 41, dtype=torch.bool, device="cuda"), 1 / (8 * f))
            close(out, want, bound_of(tol, size, vmax, want, io, cache))


@pytest.mark.parametrize("cache", CODES)
def test_attend_bad_pages_lengths_and_scales(cache):
    g = gen(14)
    c = Cache(g, 6, 2, 16, 64, cache)
    table = i32([[0, 1, -1], [2, 6, 3], [4, 5, 0], [5, 7, 9]])
    q = randn(g, 4, 4, 64, kind="bf16")

    def run(lens, window=0):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lse = torch.empty(4, 4, device="cuda")
        o = c.kv.attend(q, table, i32(lens), lse=lse, status=status, window=window)
        nan = torch.isnan(o).flatten(1)
        assert torch.equal(nan.all(1), nan.any(1)) and torch.equal(nan.all(1), torch.isnan(lse).all(1))
        return nan.all(1).tolist(), int(status)
    assert run([32, 16, 48, 0]) == ([False, False, False, False], 0)
    assert run([33, 17, 48, 16]) == ([True, True, False, False], STATUS_PAGE)
    assert run([32, 48, 49, 1]) == ([False, True, True, False], STATUS_PAGE | STATUS_POSITION)
    assert run([32, 48, 2, 1], window=16) == ([False, False, False, False], 0)
    c.scales[0][1, 0, 3] = math.nan  # one key of row 0's first kv head
    o = c.kv.attend(q, table, i32([32, 16, 48, 0]))
    assert bool(torch.isnan(o[0, :2]).all()) and not bool(torch.isnan(o[0, 2:]).any()) and not bool(torch.isnan(o[1:]).any())


def test_offsets_past_32_bits():
    pages, page, dim = 1100, 32, 128
    stride = 1 << 23  # bytes between pages: page 513 starts past 2^32
    store = torch.empty(pages * stride, dtype=torch.int8, device="cuda")
    k_pool = store.as_strided((pages, 1, page, dim), (stride, page * dim, dim, 1))
    v_pool = store.as_strided((pages, 1, page, dim), (stride, page * dim, dim, 1), storage_offset=page * dim)
    scales = store[2 * page * dim:].view(torch.float32)[: (pages - 1) * stride // 4 + 2 * page]
    ks = scales.as_strided((pages, 1, page), (stride // 4, page, 1), storage_offset=2 * page * dim // 4)
    vs = scales.as_strided((pages, 1, page), (stride // 4, page, 1), storage_offset=2 * page * dim // 4 + page)
    g = gen(15)
    use = i32([[1025, 3, 1099, 1024]])
    k, v = randn(g, 100, 1, dim), randn(g, 100, 1, dim)
    kv = PagedKV(k_pool, v_pool, ks, vs)
    at, seq = torch.arange(100, dtype=torch.int32, device="cuda"), torch.zeros(100, dtype=torch.int32, device="cuda")
    kv.append(k, v, use, at, seq=seq)
    (kc, kf), (vc, vf) = quantise(k, "i8"), quantise(v, "i8")
    assert torch.equal(k_pool[1099, 0, 5], kc[69, 0]) and torch.equal(v_pool[1024, 0, 3], vc[99, 0]) and ks[1099, 0, 5] == kf[69, 0]
    rk, rv = kv.read(use, at, seq=seq, dtype=torch.float32)
    assert torch.equal(rk, kc.float() * kf[..., None]) and torch.equal(rv, vc.float() * vf[..., None])
    q = randn(g, 1, 4, dim, kind="f16")
    o = kv.attend(q, use, i32([100]))
    w = torch.softmax(q[0].double() @ rk[:, 0].double().T / dim ** 0.5, -1)
    assert float((o[0].double() - w @ rv[:, 0].double()).abs().max()) < 4e-3  # |o| < 4 at 2^-11


def test_refusals_and_calls_without_tokens():
    g = gen(20)
    c = Cache(g, 2, 2, 16, 64, "i8")
    kv, table, lens = c.kv, torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    f = Cache(g, 2, 2, 16, 64, "bf16")
    q = randn(g, 3, 8, 64, kind="bf16")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    bad = [
        lambda: PagedKV(*c.pools), lambda: PagedKV(*c.pools, c.scales[0]), lambda: PagedKV(*f.pools, *c.scales),
        lambda: PagedKV(*c.pools, c.scales[0].double(), c.scales[1].double()),
        lambda: PagedKV(*c.pools, c.scales[0][:1], c.scales[1][:1]), lambda: PagedKV(*c.pools, c.scales[0], c.scales[1].cpu()),
        lambda: PagedKV(*c.pools, c.scales[0], c.scales[1].transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: kv.attend(q.to(torch.int8), table, lens), lambda: kv.attend(q.double(), table, lens),
        lambda: kv.read(table, lens, dtype=torch.int8), lambda: f.kv.read(table, lens, dtype=torch.float16),
        lambda: f.kv.read(table, lens, k=q[:, :2].half()), lambda: kv.read(table, lens, k=q), lambda: kv.read(table, lens.long()),
        lambda: kv.read(table, lens, seq=lens[:2]), lambda: kv.append(q[:, :2], q[:, :2], table, lens, slot=lens[:2]),
        lambda: kv.append(q[:, :2], q[:, :2], table, lens, slot=lens.long()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print(i)
    with pytest.raises(Gpt2qError, match="overlap"):
        kv.read(table, lens, k=q[:, :1].expand(-1, 2, -1))
    with pytest.raises(Gpt2qError, match="table rows"):
        kv.read(table, torch.zeros(4, dtype=torch.int32, device="cuda"))
    shared = PagedKV(*c.pools, *(s[:, :, :1].expand(-1, -1, 16) for s in c.scales))
    with pytest.raises(Gpt2qError, match="overlap"):
        shared.append(q[:, :2], q[:, :2], table, lens)
    wide = Cache(g, 2, 2, 16, 72, "f32")
    with pytest.raises(Gpt2qError, match="multiple of 16"):
        PagedKV(*(torch.zeros(2, 2, 16, 72, dtype=torch.int8, device="cuda") for _ in range(2)), *c.scales).attend(randn(g, 3, 2, 72), table, lens)
    assert wide.kv.attend(randn(g, 3, 2, 72), table, lens).shape == (3, 2, 72)
    z = torch.empty(0, 2, 64, device="cuda")
    for t in (table, table[:0]):
        kv.append(z, z, t, none)
        assert [x.shape for x in kv.read(t, none)] == [(0, 2, 64)] * 2
    assert kv.attend(torch.empty(0, 8, 64, device="cuda"), table[:0], none).shape == (0, 8, 64)


def test_captured_and_replayed_on_other_streams():
    """Append, read and attend captured together, twice; replayed at once on two streams over caches of their own."""
    g = gen(17)
    rot = Rotary(128)
    sets = []
    for s in range(2):
        c = Cache(gen(100 + s), 40, 2, 16, 128, CODES[s])
        d = dict(c=c, table=torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20), lens=i32([200, 31]), pos=i32([199, 30]),
                 qkv=randn(g, 2, 12, 128, kind="bf16"))
        sets.append(d)

    def step(d):
        q = d["c"].kv.append(d["qkv"][:, 8:10], d["qkv"][:, 10:], d["table"], d["pos"], rotary=rot, q=d["qkv"][:, :8])
        return [d["c"].kv.attend(q, d["table"], d["lens"]), *d["c"].kv.read(d["table"], d["pos"])]
    step(sets[0]), step(sets[1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    torch.cuda.synchronize()
    for d, st in zip(sets, streams):
        with torch.cuda.stream(st):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=st):
                out = step(d)
        graphs.append((gr, out))
    for at in ([5, 0], [319, 318]):
        for d in sets:
            d["pos"].copy_(i32(at)), d["lens"].copy_(i32(at) + 1), d["qkv"].copy_(randn(g, 2, 12, 128, kind="bf16"))
        torch.cuda.synchronize()
        for st, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for d, (_, out) in zip(sets, graphs):
            got = [x.clone() for x in out]
            for a, b in zip(got, step(d)):
                assert torch.equal(a, b)
