"""Token log probabilities of a few long rows, each of which a cluster of 2 to 8 blocks shares: the form without
alternatives against the form with one, and against 64 bits.

Tolerance: test_gpu_logprobs derives it (d = (V / 256 + 64) 2^-24 + 2^-18 for the sums of V terms)."""
import math

import pytest
import torch

from smelt_b200.logprobs import token_logprobs, token_logprobs_grad

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def delta(vocab):
    return (vocab / 256 + 64) * 2.0 ** -24 + 2.0 ** -18


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("vocab", [8193, 50257])
@pytest.mark.parametrize("rows", [1, 2, 74, 75, 148, 149, 296, 297])
def test_without_alternatives(kind, vocab, rows):
    """Calls that follow one another without a pause, so that blocks of the next cluster start while others still run."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.empty(rows, vocab, dtype=T[kind], device="cuda").normal_(0, 2.5, generator=g)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    got = [token_logprobs(x, t) for _ in range(20)]
    one = token_logprobs(x, t, top=1)
    for r in got:
        assert torch.equal(r.lp, one.lp) and torch.equal(r.entropy, one.entropy) and torch.equal(r.stats, one.stats)
    lp = torch.log_softmax(x.double(), 1)
    h = torch.special.entr(lp.exp()).sum(1)
    want = lp.gather(1, t[:, None])[:, 0]
    d = delta(vocab)
    assert bool(((one.lp.double() - want).abs() <= 2.0 ** -22 * (want.abs() + 16) + d).all())
    assert bool(((one.entropy.double() - h).abs() <= 2 * d * (1 + 2 * h)).all())


@pytest.mark.parametrize("temperature", [1.01e-30, 1e-20, 1e30])
def test_extreme_temperatures(temperature):
    """Almost 0: all of the probability on the largest logit, nothing else. Very high: all alike."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(2, 300, device="cuda").normal_(0, 3, generator=g)
    best = x.argmax(1)
    r = token_logprobs(x, best, top=3, temperature=temperature)
    assert torch.equal(r.top_ids[:, 0].long(), best)
    want = 0.0 if temperature < 1 else -math.log(300)
    assert bool(((r.lp - want).abs() < 1e-5).all()) and bool(((r.entropy + want).abs() < 1e-5).all())
    d = token_logprobs_grad(x, best, r.stats, torch.ones(2, device="cuda"), torch.ones(2, device="cuda"), temperature=temperature)
    assert bool(torch.isfinite(d).all())


@pytest.mark.parametrize("kind", list(T))
@pytest.mark.parametrize("rows", [1, 3, 40, 148, 300, 600])
@pytest.mark.parametrize("top", [1, 20, 21, 64])
def test_alternatives_that_lie_together(kind, rows, top):
    """A contiguous range of the vocabulary is allowed, from a few tokens to thousands, at its beginning, middle or end; and a
    vocabulary ordered by frequency."""
    vocab = 50257
    g = torch.Generator(device="cuda").manual_seed(rows + top)
    base = torch.empty(rows, vocab, device="cuda").normal_(0, 2.5, generator=g)
    for low, high in ((0, 6000), (0, 5), (31_000, 33_100), (49_000, vocab), (20_000, 20_500), (7, 9000)):
        x = torch.full_like(base, -math.inf)
        x[:, low:high] = base[:, low:high]
        x = x.to(T[kind])
        r = token_logprobs(x, top=top)
        ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(r.top_ids.long(), ids), (low, high)
    x = (base * 0.2 - 6 * torch.log1p(torch.arange(vocab, device="cuda") / 100.0)).to(T[kind])
    r = token_logprobs(x, top=top)
    lp = torch.log_softmax(x.double(), 1)
    ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.top_ids.long(), ids)
    want = lp.gather(1, ids)
    assert bool(((r.top_lp.double() - want).abs() <= 2.0 ** -22 * (want.abs() + 16) + delta(vocab)).all())


@pytest.mark.parametrize("kind", list(T))
def test_gradient_beside_its_logits_in_one_buffer(kind):
    """Logits and gradient side by side in the rows of one buffer; one shifted over the other is refused."""
    from smelt_b200._ffi import Gpt2qError

    g = torch.Generator(device="cuda").manual_seed(5)
    buf = torch.empty(9, 2 * 1003, dtype=T[kind], device="cuda").normal_(0, 2, generator=g)
    x, dx = buf[:, :1003], buf[:, 1003:]
    t = torch.randint(0, 1003, (9,), generator=g, device="cuda")
    d = torch.empty(9, device="cuda").normal_(generator=g)
    r = token_logprobs(x, t)
    want = token_logprobs_grad(x.contiguous(), t, r.stats, d, d)
    keep = x.clone()
    token_logprobs_grad(x, t, r.stats, d, d, out=dx)
    assert torch.equal(dx, want) and torch.equal(x, keep)
    for out in (buf[:, 1:1004], buf[:, 1002:2005]):
        with pytest.raises(Gpt2qError, match="overlap"):
            token_logprobs_grad(x, t, r.stats, d, d, out=out)
    with pytest.raises(Gpt2qError, match="overlap"):
        token_logprobs_grad(x[:8], t[:8], r.stats[:8], d[:8], d[:8], out=x[1:])
    assert torch.equal(x, keep)
