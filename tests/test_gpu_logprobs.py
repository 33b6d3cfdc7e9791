"""Token log probabilities on the GPU (smelt_b200.logprobs) against a plain implementation in 64 bits.

Tolerances, derived before the first run, with u = 2^-24:
 z = (x - m) / t carries 3 u |z|; exp adds 2^-22 and its argument's error. A sum of V terms runs in strips of at
 most V / 256 + 64 additions: d = (V / 256 + 64) u + 16 * 2^-22 bounds the relative error of S and of sum e|z|, as the
 probability-weighted |z| is at most ln V + 1 < 16 beside ln S. So ln p: 2^-22 (|z| + 1) + d; entropy: 2 d (1 + H + |ln S|).
 Gradient: p within (|ln p| + 16) 2^-21 + d relative, both terms; plus the output's rounding."""
import math

import numpy as np
import pytest
import torch

from smelt_b200.logprobs import TOP_MAX, token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def make(seed, rows, vocab, kind, scale=2.5, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, vocab + pad, dtype=T[kind], device="cuda").normal_(0, scale, generator=g)[:, :vocab]
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    return x, t


def delta(vocab):
    return (vocab / 256 + 64) * 2.0 ** -24 + 16 * 2.0 ** -22


def check(x, t, top=0, temperature=1.0):
    rows, vocab = x.shape
    r = token_logprobs(x, t, top=top, temperature=temperature)
    y = x.double() / temperature
    lp = torch.log_softmax(y, 1)
    p = lp.exp()
    h = torch.special.entr(p).sum(1)
    m = y.amax(1)
    d = delta(vocab)
    ls = torch.logsumexp(y - m[:, None], 1)
    want = lp.gather(1, t.long().clamp(0)[:, None])[:, 0]
    want = torch.where(t < 0, torch.zeros_like(want), want)
    z = (y - m[:, None]).abs()
    zt = z.gather(1, t.long().clamp(0)[:, None])[:, 0]
    same = torch.isinf(want)
    assert torch.equal(r.lp[same].double(), want[same])
    assert bool(((r.lp.double() - want).abs() <= 2.0 ** -22 * (zt + 1) + d)[~same].all())
    assert bool(((r.entropy.double() - h).abs() <= 2 * d * (1 + h + ls)).all())
    assert torch.equal(r.stats[:, 0], x.float().amax(1)) and torch.equal(r.stats[:, 2], r.entropy)
    assert bool(((r.stats[:, 1].double() - ls).abs() <= d * (1 + ls)).all())
    if top:
        order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids.long(), order)
        want = lp.gather(1, order)
        lim = 2.0 ** -22 * (z.gather(1, order) + 1) + d
        inf = torch.isinf(want)
        assert torch.equal(r.top_lp[inf].double(), want[inf])
        assert bool(((r.top_lp.double() - want).abs() <= lim)[~inf].all())
    else:
        assert r.top_ids is None and r.top_lp is None
    return r


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("rows,vocab,top,pad", [(1, 1, 1, 0), (1, 50257, 5, 0), (3, 97, 20, 3), (2, 64, 64, 0), (7, 4097, 64, 1),
                                                (33, 1031, 8, 5), (2, 200003, 20, 0), (300, 257, 1, 0), (5, 31, 0, 2)])
def test_matches_definition(kind, rows, vocab, top, pad):
    x, t = make(1, rows, vocab, kind, pad=pad)
    check(x, t, top)
    check(x, t.to(torch.int32), min(top, 3), temperature=0.7)


@pytest.mark.parametrize("kind", list(T))
def test_unaligned_rows_and_high_temperature(kind):
    g = torch.Generator(device="cuda").manual_seed(2)
    flat = torch.empty(5 * 1001 + 1, dtype=T[kind], device="cuda").normal_(0, 4, generator=g)
    x = flat[1:].view(5, 1001)
    t = torch.tensor([0, 1000, 5, -1, -7], device="cuda")
    check(x, t, 9, temperature=3.0)


@pytest.mark.parametrize("vocab", [100, 50257])
@pytest.mark.parametrize("shape", ["equal", "rising", "falling", "one", "pairs", "blocks"])
def test_ties_and_orders(vocab, shape):
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"equal": i * 0, "rising": i * 1e-3, "falling": -i * 1e-3, "one": torch.where(i == vocab - 3, 5.0, 0.0),
           "pairs": (i // 2) * 1e-2, "blocks": torch.floor(i / 4096) * 0.5}[shape]
    x = torch.stack([row, row.flip(0)])
    t = torch.tensor([0, vocab - 1], device="cuda")
    for top in (1, 20, 64):
        check(x, t, top)
    check(x.to(torch.bfloat16), t, 20)


@pytest.mark.parametrize("rows,top", [(600, 20), (600, 64), (1, 20)])
def test_alternatives_crowded_into_few_threads(rows, top):
    """The likeliest tokens all lie in the same few strided vectors, thousands of them above the best of the rest."""
    vocab = 50256
    lane = (torch.arange(vocab, device="cuda") // 4) % 128
    g = torch.Generator(device="cuda").manual_seed(14)
    x = torch.empty(rows, vocab, device="cuda").normal_(0, 0.1, generator=g) - lane
    check(x, torch.zeros(rows, dtype=torch.int64, device="cuda"), top)


def test_signed_zeros_tie():
    x = torch.full((1, 3000), -1.0, device="cuda")
    x[0, 5], x[0, 2000] = -0.0, 0.0
    assert token_logprobs(x, top=2).top_ids.tolist() == [[5, 2000]]


@pytest.mark.parametrize("kind", list(T))
def test_masked_logits(kind):
    """-inf on most of the vocabulary, the type's lowest value elsewhere; more alternatives asked than remain."""
    x, _ = make(3, 4, 5000, kind)
    x[0, 7:] = -math.inf          # seven tokens left
    x[1, 1:] = -math.inf          # one token left: probability 1
    x[2, :4990] = torch.finfo(T[kind]).min
    x[3, ::2] = -math.inf
    t = torch.tensor([3, 0, 4995, 4], device="cuda")
    r = check(x, t, 20)
    assert float(r.lp[1]) == 0.0 and float(r.entropy[1]) == 0.0
    assert float(r.lp[3]) == -math.inf
    assert bool(torch.isneginf(r.top_lp[0, 7:]).all()) and r.top_ids[0, 7:].tolist() == list(range(7, 20))
    low = torch.full((1, 300), torch.finfo(T[kind]).min, dtype=T[kind], device="cuda")
    r = token_logprobs(low, torch.tensor([9], device="cuda"), top=2, temperature=0.5)
    assert abs(float(r.lp) + math.log(300)) < 1e-5 and r.top_ids.tolist() == [[0, 1]]


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("vocab", [40, 50257])
def test_empty_nan_and_infinite_rows(kind, vocab):
    x, _ = make(4, 5, vocab, kind)
    x[0] = -math.inf
    x[2, 11] = math.nan
    x[3, 13] = math.inf
    t = torch.tensor([1, 2, 3, 4, vocab], device="cuda")
    d = torch.ones(5, device="cuda")
    r = token_logprobs(x, t, top=4)
    assert float(r.lp[0]) == -math.inf and float(r.entropy[0]) == 0.0
    assert r.top_ids[0].tolist() == [0, 1, 2, 3] and bool(torch.isneginf(r.top_lp[0]).all())
    for bad in (2, 3):
        assert math.isnan(float(r.lp[bad])) and math.isnan(float(r.entropy[bad])) and bool(torch.isnan(r.top_lp[bad]).all())
    assert int(r.top_ids[3, 0]) == 13 and 11 not in r.top_ids[2].tolist()
    assert math.isnan(float(r.lp[4])) and math.isfinite(float(r.entropy[4]))  # a target past the vocabulary
    check(x[1:2], t[1:2], 4)
    gr = token_logprobs_grad(x, t, r.stats, d, d)
    assert bool((gr[0] == 0).all()) and bool(torch.isfinite(gr[1]).all())
    for bad in (2, 3, 4):
        assert bool(torch.isnan(gr[bad]).any())
    only = torch.full((1, vocab), math.nan, dtype=T[kind], device="cuda")
    assert token_logprobs(only, top=3).top_ids.tolist() == [[0, 1, 2]]


# ------------------------------------------------------------------------------------- gradient
def grad64(x, t, g, ge, temperature):
    lp = torch.log_softmax(x.double() / temperature, 1)
    p = lp.exp()
    h = torch.special.entr(p).sum(1, keepdim=True)
    lps = torch.where(p > 0, lp, torch.zeros_like(lp))
    d = torch.zeros_like(p)
    size = torch.zeros_like(p)
    if g is not None:
        gd = torch.where(t < 0, torch.zeros_like(g), g).double()[:, None]
        d = -gd * p
        d.scatter_add_(1, t.long().clamp(0)[:, None], gd)
        size = gd.abs() * p
    if ge is not None:
        d = d - ge.double()[:, None] * p * (lps + h)
        size = size + ge.double().abs()[:, None] * p * (1 + lps.abs() + h)
    rel = (lps.abs() + 16) * 2.0 ** -21 + delta(x.shape[1])
    e = torch.finfo(x.dtype).eps / 2
    step = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}[x.dtype]
    return d / temperature, size / temperature * 2 * rel + d.abs() / temperature * (e * 1.01 + 2.0 ** -22) + step * 4


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (2, 97, 0), (64, 1031, 9), (3, 50257, 0), (5, 4096, 0), (1, 200003, 0)])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_gradient_matches_formula(kind, rows, vocab, pad, temperature):
    x, t = make(5, rows, vocab, kind, pad=pad)
    if rows > 1:
        t[1] = -1
        x[0, 1:vocab // 2] = -math.inf
        t[0] = 0
    g = torch.Generator(device="cuda").manual_seed(6)
    dl, de = (torch.empty(rows, device="cuda").normal_(0, 1, generator=g) for _ in range(2))
    stats = token_logprobs(x, t, temperature=temperature).stats
    for a, b in ((dl, None), (None, de), (dl, de)):
        got = token_logprobs_grad(x, None if a is None else t, stats, a, b, temperature=temperature)
        want, tol = grad64(x, t, a, b, temperature)
        assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() - tol).max())


@pytest.mark.parametrize("kind", list(T))
def test_gradient_in_place_and_into_a_padded_output(kind):
    x, t = make(7, 6, 1003, kind, pad=5)
    d = torch.linspace(-1, 1, 6, device="cuda")
    stats = token_logprobs(x, t).stats
    want = token_logprobs_grad(x, t, stats, d, d)
    hold = torch.full((6, 1010), 3.0, dtype=T[kind], device="cuda")
    out = hold[:, 3:1006]
    assert token_logprobs_grad(x, t, stats, d, d, out=out) is out
    assert torch.equal(out, want) and bool((hold[:, :3] == 3).all()) and bool((hold[:, 1006:] == 3).all())
    tail = x.as_strided((6, 5), (1008, 1), storage_offset=1003).clone()
    token_logprobs_grad(x, t, stats, d, d, out=x)
    assert torch.equal(x, want) and torch.equal(x.as_strided((6, 5), (1008, 1), storage_offset=1003), tail)


def test_gradient_matches_differences():
    """Central differences with h = 1/32: the truncation h^2 / 6 |f'''| is under 6.6e-4 (|f'''| < 4 for the
    temperature's 1 / 0.8 cubed), the forward's rounding under 4e-6 / (2 h) = 6.4e-5."""
    x, t = make(8, 1, 12, "f32", scale=1.0)
    g, ge, h = 1.3, -0.7, 1 / 32
    gd, hd = torch.tensor([g], device="cuda"), torch.tensor([ge], device="cuda")
    got = token_logprobs_grad(x, t, token_logprobs(x, t, temperature=0.8).stats, gd, hd, temperature=0.8)[0]
    for j in range(12):
        f = []
        for s in (h, -h):
            y = x.clone()
            y[0, j] += s
            r = token_logprobs(y, t, temperature=0.8)
            f.append(g * float(r.lp) + ge * float(r.entropy))
        assert abs((f[0] - f[1]) / (2 * h) - float(got[j])) < 2 * (6.6e-4 + 6.4e-5)


def test_rows_past_32_bit_offsets():
    """Row starts past 2^31 elements."""
    rows, ld = 3, 1_200_000_000
    store = torch.empty(2 * ld + 1000, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((rows, 1000), (ld, 1))
    small, t = make(9, rows, 1000, "bf16")
    x.copy_(small)
    a, b = token_logprobs(x, t, top=5), token_logprobs(small, t, top=5)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    d = torch.ones(rows, device="cuda")
    want = token_logprobs_grad(small, t, b.stats, d, d)
    token_logprobs_grad(x, t, a.stats, d, d, out=x)
    assert torch.equal(x, want)


def test_deterministic_captured_and_replayed():
    x, t = make(10, 9, 50257, "bf16")
    d = torch.ones(9, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            r = token_logprobs(x, t, top=20)
            dx = token_logprobs_grad(x, t, r.stats, d, d)
    torch.cuda.synchronize()
    for seed in (11, 12):
        y, u = make(seed, 9, 50257, "bf16")
        x.copy_(y)
        t.copy_(u)
        want = token_logprobs(x, t, top=20)
        again = token_logprobs(x, t, top=20)
        wd = token_logprobs_grad(x, t, want.stats, d, d)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(r, want)) and all(torch.equal(a, b) for a, b in zip(again, want))
        assert torch.equal(dx, wd)


def test_no_rows():
    x = torch.empty(0, 50, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    r = token_logprobs(x, t, top=3)
    assert r.lp.shape == (0,) and r.top_ids.shape == (0, 3)
    assert token_logprobs_grad(x, t, r.stats, torch.empty(0, device="cuda")).shape == (0, 50)
    assert TOP_MAX == 64
