"""Attention over paged caches where every warp streams many tiles: ring refills, runs inside a row, long sums.

Rows are long and name the pages of a small pool many times over, so that a reference in 64 bits needs only how often
each slot counts.

Tolerance of an output, with u = 2^-24, weights w_k = softmax(s)_k and o the result. A weight is off by the factor 1 + e_k:
 * the score: 16-bit caches take dim / 16 matrix steps, each of which may round its running sum (at most
   S_k = scale sum |q_i k_ki|) down by 2 u: dim / 8 u S_k, and 8 u S_k for its pieces' sums; on fp32 caches two or more lanes
   share a key's chain of fused multiply-adds: dim / 2 u S_k + 8 u S_k;
 * the exponent's argument, its factor and ex2 (2 ulp), and up to 12 changes of the running maximum and joins:
   (2 |s_k - max| + 24) 2 u.
 The output moves by sum w_k e_k (|v_k| + |o|). The sums over a warp's n tiles round once a tile (fp32 caches: once a key), the
 pieces of a tile and the joins of at most 12 warps and 32 lanes add 80: (n + 80) u sum w_k |v_k|, and half of that for the sum
 of weights times |o|. The type's rounding comes last. The logarithm of the sum is off by sum w_k e_k + (n + 80) u and its own
 rounding, 4 u (|lse| + 1)."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]
BLOCKS, WARPS = 148, 12  # the most that a call runs


def tile_keys(cache, dim):
    """Keys of a tile: 4 KB of keys, and at least 8 (fp32) or 16."""
    hd = 64 if dim <= 64 else 128 if dim <= 128 else 256
    size = 4 if cache == "f32" else 2
    return max(4096 // (hd * size), 8 if cache == "f32" else 16)


def tiles_per_warp(lens, window, kv, cache, dim):
    keys = [min(n, window) if window else n for n in lens]
    return sum(-(-n // tile_keys(cache, dim)) for n in keys) * kv / (BLOCKS * WARPS)


def counts(table, lens, window, page, slots):
    """How often each slot of the pool counts for every row, [rows, slots]."""
    out = torch.zeros(len(lens), slots, dtype=torch.float64, device=table.device)
    for r, n in enumerate(lens):
        j = torch.arange(max(0, n - window) if window else 0, n, device=table.device)
        at = table[r, torch.div(j, page, rounding_mode="floor")].long() * page + j % page
        out[r] = torch.bincount(at, minlength=slots).double()
    return out


def reference(q, k_pool, v_pool, count, cache, io, n):
    """(out, its tolerance, lse, its tolerance) for slots that count `count` times; n: roundings of a running sum."""
    rows, heads, dim = q.shape
    kv = k_pool.shape[1]
    scale = dim ** -0.5
    K, V = (x.double().transpose(1, 2).reshape(-1, kv, dim) for x in (k_pool, v_pool))
    Q = q.double().view(rows, kv, heads // kv, dim)
    s = torch.einsum("rhgd,khd->rhgk", Q, K) * scale
    mag = torch.einsum("rhgd,khd->rhgk", Q.abs(), K.abs()) * scale
    s = s.masked_fill((count == 0)[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = count[:, None, None] * torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    w = e / total.clamp(min=1e-300)
    o = torch.einsum("rhgk,khd->rhgd", w, V)
    steps = dim / (2 if cache == "f32" else 8) + 8
    eps = steps * U * mag + (2 * (s - m).abs().nan_to_num(posinf=0.0) + 24) * 2 * U
    we = w * eps
    va = torch.einsum("rhgk,khd->rhgd", w, V.abs())
    tol = torch.einsum("rhgk,khd->rhgd", we, V.abs()) + we.sum(-1, keepdim=True) * o.abs() + (n + 80) * U * (va + o.abs() / 2)
    half = torch.finfo(T[io]).eps / 2
    tol = tol + o.abs() * half * 1.01 + (2.0 ** -25 if io == "f16" else 0)
    lse = (m + torch.log(total))[..., 0]
    ltol = we.sum(-1) + (n + 80) * U + 4 * U * (lse.abs().nan_to_num(posinf=0.0) + 1)
    shape = (rows, heads, dim)
    return o.reshape(shape), tol.reshape(shape), lse.reshape(rows, heads), ltol.reshape(rows, heads)


# dim, kv heads, query heads per kv head, page, lens, window. Pages of 21 slots are gathered key by key.
CASES = [
    (64, 8, 2, 64, [40000, 3, 17001, 0, 16100], 0),
    (64, 8, 1, 21, [60000, 17, 25001], 50000),
    (80, 4, 5, 48, [80011, 1], 0),
    (128, 8, 4, 64, [30001, 0, 6000], 0),
    (128, 4, 16, 16, [71999], 0),
    (128, 8, 2, 21, [5, 26000, 40000], 17000),
    (192, 4, 3, 32, [71500, 129], 0),
    (256, 4, 2, 16, [65000, 300, 7000], 0),
    (256, 4, 8, 21, [77000], 71500),
]


def make(seed, case, io, cache, device):
    dim, kv, group, page, lens, _ = case
    pages = max(8, 4096 // page)
    rng = np.random.default_rng(seed)
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape, kind):
        return torch.empty(shape, dtype=T[kind], device=device).normal_(0, 1, generator=g)
    k, v = (randn(pages, kv, page, dim, kind=cache) for _ in range(2))
    table = torch.from_numpy(rng.integers(0, pages, (len(lens), -(-max(lens) // page))).astype(np.int32)).to(device)
    return k, v, randn(len(lens), kv * group, dim, kind=io), table


def roundings(case, cache):
    """Of a warp's running sum: with half as many warps as a call can run, whatever the tile's size."""
    dim, kv, _, _, lens, window = case
    n = 2 * tiles_per_warp(lens, window, kv, cache, dim) + 1
    return n * tile_keys(cache, dim) if cache == "f32" else n


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_many_tiles_per_warp(case, io, cache):
    from smelt_b200.paged import PagedKV

    dim, kv, group, page, lens, window = case
    assert tiles_per_warp(lens, window, kv, cache, dim) >= 9
    k, v, q, table = make(3, case, io, cache, "cuda")
    count = counts(table, lens, window, page, k.shape[0] * page)
    want, tol, wlse, ltol = reference(q, k, v, count, cache, io, roundings(case, cache))
    lse = torch.empty(q.shape[:2], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = PagedKV(k, v).attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window, lse=lse, status=status)
    assert int(status) == 0
    empty = torch.tensor([n == 0 for n in lens], device="cuda")
    assert bool((out[empty] == 0).all()) and bool(torch.isneginf(lse[empty]).all())
    over = (out.double() - want).abs() - tol
    assert float(over[~empty].max()) <= 0, (float(over[~empty].max()), float(tol[~empty].max()))
    over = (lse.double() - wlse).abs() - ltol
    assert float(over[~empty].max()) <= 0, (float(over[~empty].max()), float(ltol[~empty].max()))


@pytest.mark.parametrize("case", [c for c in CASES if c[0] in (64, 128) and c[2] < 16], ids=str)
@pytest.mark.parametrize("io,cache", [("f32", "f16"), ("bf16", "bf16"), ("f32", "f32")])
def test_the_tolerance_notices_a_tile(case, io, cache):
    """A tile that is left out or counted twice moves the result past the tolerance (planted in the reference)."""
    dim, kv, group, page, lens, window = case
    case = (dim, 1, 1, page, lens, window)  # one head is enough
    k, v, q, table = make(4, case, io, cache, "cpu")
    n = roundings((dim, kv, group, page, lens, window), cache)
    slots = k.shape[0] * page
    count = counts(table, lens, window, page, slots)
    want, tol, wlse, ltol = reference(q, k, v, count, cache, io, n)
    tk = tile_keys(cache, dim)
    rng = np.random.default_rng(5)
    for r, ln in enumerate(lens):
        lo = max(0, ln - window) if window else 0
        for _ in range(3 if ln > tk else 0):
            j = torch.arange(tk) + int(rng.integers(lo, ln - tk) // tk * tk)
            j = j[j >= lo]
            at = table[r, torch.div(j, page, rounding_mode="floor")].long() * page + j % page
            for sign in (1, -1):
                planted = count.clone()
                planted[r] += sign * torch.bincount(at, minlength=slots).double()
                o, _, l, _ = reference(q, k, v, planted, cache, io, n)
                assert bool((((o - want).abs() > tol)[r]).any()) or bool(((l - wlse).abs() > ltol)[r].any())
                assert bool(((l - wlse).abs() > ltol)[r].all())


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_of_one_sign_do_not_drift(dim, io, cache):
    """Values of 1 everywhere: the result is 1 whatever the weights. Sums that are rounded to nearest leave a random walk:
    over n additions to a growing sum, u sqrt(n) / 3 rms, for numerator and denominator; six of them for both, 3 u sqrt(n). A
    tile's own matrix steps (at most six) round down by 2 u each: 12 u; pieces of a weight and the joins 12 u more."""
    from smelt_b200.paged import PagedKV

    kv, rows, page, pages = 4, 40, 64, 16
    keys = 110_000 if cache != "f32" else 30_000
    g = torch.Generator(device="cuda").manual_seed(6)
    k = torch.empty(pages, kv, page, dim, dtype=T[cache], device="cuda").normal_(0, 1, generator=g)
    v = torch.ones_like(k)
    q = torch.empty(rows, kv, dim, dtype=T[io], device="cuda").normal_(0, 1, generator=g)
    width = -(-keys // page)
    table = torch.randint(0, pages, (rows, width), generator=g, device="cuda").to(torch.int32)
    lens = [keys - 7 * r for r in range(rows)]
    out = PagedKV(k, v).attend(q, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    n = 2 * tiles_per_warp(lens, 0, kv, cache, dim) * (tile_keys(cache, dim) if cache == "f32" else 1)
    assert n > 500
    off = float((out.double() - 1).abs().max())
    lim = (3 * math.sqrt(n) + 24) * U
    if io != "f32":
        lim = 0.0  # 1 is a number of the type, and the sums' error is far below half a step beside it
    assert off <= lim, (off / U, lim / U)


@pytest.mark.gpu
@pytest.mark.parametrize("io,cache", TYPES)
def test_values_that_cancel_keep_the_weights_bits(io, cache):
    """The likeliest key has the value 0; two others of almost equal score have 1 and -1, so the result is the small
    difference of their weights and shows how many bits those have. Scores and the largest weight are exact; a weight is within
    (2 a + 4) 2 u (its exponent's argument, at most a, and ex2 to 2 ulp), its pieces and their sums within 8 u, but for bf16
    tensors, whose weights take two pieces of 8 bits: 2^-16. The output's own rounding is beside the small result."""
    from smelt_b200.paged import PagedKV

    rows, dim = 64, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    k = torch.zeros(rows, 1, 3, dim, dtype=T[cache], device="cuda")
    v = torch.zeros_like(k)
    v[:, :, 1], v[:, :, 2] = 1, -1
    q = torch.zeros(rows, 1, dim, dtype=T[io], device="cuda")
    q[:, 0, 0] = 1
    q[:, 0, 1] = 2.0 ** -(torch.arange(rows, device="cuda") % 8 + 5).float()
    k[:, 0, 1:, 0] = torch.empty(rows, 1, device="cuda").uniform_(-0.7, -0.1, generator=g).to(T[cache])
    k[:, 0, 2, 1] = -1
    table = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None]
    out = PagedKV(k, v).attend(q, table, torch.full((rows,), 3, dtype=torch.int32, device="cuda"), scale=1.0)
    s1 = k[:, 0, 1, 0].double()
    w1, w2 = torch.exp(s1), torch.exp(s1 - q[:, 0, 1].double())
    total = 1 + w1 + w2
    want = ((w1 - w2) / total)[:, None]
    pieces = 2.0 ** -16 if io == "bf16" else 8 * U
    tol = ((w1 + w2) / total)[:, None] * ((2 * 0.75 + 4) * 2 * U + pieces) + want.abs() * (torch.finfo(T[io]).eps / 2) * 1.01
    err = (out[:, 0].double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
