"""The model over the operators on device memory: gpt2q_score against the oracle's logits, gpt2q_trunk_score_grad
against the oracle's backward, and decode over paged caches against the arena's decode.

Tolerances: the logits are within `observed` of the oracle's (the handle's own guard, e = 1e-3 by default). ln p moves by
at most 2 e; an entropy by e * sum p |ln p + H| <= 2 e H."""
import numpy as np
import pytest
import torch

from oracle import backward_oracle as B
from smelt_b200._ffi import Gpt2qError
from smelt_b200.gpu import Gpu
from smelt_b200.logprobs import token_logprobs
from smelt_b200.paged import PagedKV

from .helpers import MINI, TINY, make_pack, observed, oracle_engine, oracle_prefix_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def log_softmax64(x):
    x = x.astype(np.float64)
    z = x - x.max(-1, keepdims=True)
    return z - np.log(np.exp(z).sum(-1, keepdims=True))


@pytest.mark.parametrize("meta,policy", [(TINY, "auto"), (MINI, "auto"), (MINI, "q4auto"), (TINY, "f32")])
def test_score_matches_oracle_and_nll(meta, policy):
    pk = make_pack(meta, policy, 0, 0.02)
    eng = oracle_engine(pk)
    ids = np.random.default_rng(3).integers(0, meta.vocab, meta.n_ctx).astype(np.uint32)
    with Gpu(pk, max_seqs=2) as g:
        e = observed(g)
        for n in (2, 9, meta.n_ctx):
            lp, ent, top_ids, top_lp = g.score(ids[:n], top=7, slot=1)
            ref = log_softmax64(oracle_prefix_logits(eng, ids[: n - 1]))
            assert np.abs(lp - ref[np.arange(n - 1), ids[1:n]]).max() <= 2 * e
            h = -(np.exp(ref) * ref).sum(-1)
            assert np.all(np.abs(ent - h) <= 2 * e * h + 1e-5)
            assert np.all(np.diff(top_lp, axis=1) <= 0) and all(len(set(r)) == 7 for r in top_ids.tolist())
            assert np.abs(top_lp - np.take_along_axis(ref, top_ids.astype(np.int64), 1)).max() <= 2 * e
            assert np.abs(top_lp - -np.sort(-ref, 1)[:, :7]).max() <= 2 * e
            assert abs(-lp.astype(np.float64).mean() - g.nll(ids[:n])) < 1e-5  # fp32 rounding of each term
        lp0, _, i0, _ = g.score(ids[:5])
        assert i0.shape == (4, 0) and np.array_equal(lp0, g.score(ids[:5], top=1)[0])


def test_score_refusals():
    pk = make_pack(TINY, "auto")
    with Gpu(pk) as g:
        ids = np.arange(5, dtype=np.uint32)
        for bad in (dict(top=-1), dict(top=65), dict(slot=1), dict(slot=-1)):
            with pytest.raises(Gpt2qError):
                g.score(ids, **bad)
        with pytest.raises(Gpt2qError):
            g.score(ids[:1])
        with pytest.raises(Gpt2qError, match="vocab"):
            g.score(np.array([1, TINY.vocab], np.uint32))
        assert g.score(ids)[0].shape == (4,)


@pytest.mark.parametrize("meta,policy,n", [(TINY, "auto", 9), (MINI, "auto", 33), (TINY, "f32", 64), (MINI, "q4auto", 1)])
def test_trunk_score_grad_matches_oracle(meta, policy, n):
    pk = make_pack(meta, policy, 0, 0.02)
    W = B.weights64(pk)
    rng = np.random.default_rng(5)
    ids = rng.integers(0, meta.vocab, n).astype(np.uint32)
    tgt = rng.integers(0, meta.vocab, n).astype(np.int32)
    if n > 4:
        tgt[3] = -1
    dl, de = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    logits, acts = B.forward_stash(W, meta, ids)
    lp = log_softmax64(logits)
    p = np.exp(lp)
    h = -(p * lp).sum(-1, keepdims=True)
    with Gpu(pk) as g:
        for a, b in ((dl, de), (dl, None), (None, de)):
            d = np.zeros_like(p)
            if a is not None:
                w = np.where(tgt < 0, 0.0, a.astype(np.float64))
                d -= w[:, None] * p
                d[np.arange(n), np.maximum(tgt, 0)] += w
            if b is not None:
                d -= b.astype(np.float64)[:, None] * p * (lp + h)
            dx, lnf, glp, gent = g.trunk_score_grad(ids, tgt, a, b)
            ref = B.trunk_input_grad(W, meta, acts, d)
            # the backward's own bound (test_gpu_backward) for each of the two devices' steps: logits, then trunk
            assert B.rel_max(dx, ref) < 4e-3, B.rel_max(dx, ref)
            want = np.where(tgt < 0, 0.0, lp[np.arange(n), np.maximum(tgt, 0)])
            assert np.abs(glp - want).max() <= 2e-3 and np.abs(gent - h[:, 0]).max() <= 2e-3 * max(1.0, h.max())
        # the same gradient through host dlogits
        dx2, lnf2 = g.trunk_input_grad(ids, d.astype(np.float32))
        assert B.rel_max(dx, dx2) < 4e-3 and np.array_equal(lnf, lnf2)
        with pytest.raises(Gpt2qError, match="target"):
            g.trunk_score_grad(ids, np.full(n, meta.vocab, np.int32), dl)


def caches(meta, pages, page, kind):
    hd = meta.n_embd // meta.n_head
    out = []
    for _ in range(meta.n_layer):
        k, v = (torch.full((pages, page, meta.n_head, hd), float("nan"), dtype=kind, device="cuda").transpose(1, 2) for _ in range(2))
        out.append(PagedKV(k, v))
    return out


@pytest.mark.parametrize("kind,bound", [(torch.float32, 1e-3), (torch.float16, 2e-2)])
@pytest.mark.parametrize("meta,policy,page", [(MINI, "auto", 16), (MINI, "f32", 5), (TINY, "q4auto", 64)])
def test_decode_paged_matches_the_arena(kind, bound, meta, policy, page):
    """Prefilled slots are copied to pages, then both caches decode the same tokens; fp32 pages to the arithmetic's
    accuracy, fp16 pages within the acceptance bound of the logits (they round keys and values to 2^-12)."""
    pk = make_pack(meta, policy, 0, 0.02)
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, meta.vocab, n).astype(np.uint32) for n in (5, 1, 40, 17)]
    width = -(-meta.n_ctx // page)
    table = torch.from_numpy(rng.permutation(4 * width).astype(np.int32).reshape(4, width)).cuda()
    with Gpu(pk, max_seqs=4) as g:
        layers = caches(meta, 4 * width, page, kind)
        nxt = g.prefill(prompts)
        for s, p in enumerate(prompts):
            g.page_out(s, p.size, layers, table, s)
        tok, pos = nxt.copy(), np.array([p.size for p in prompts], np.int32)
        for _ in range(6):
            a, la = g.decode(tok, pos, want_logits=True)
            b, lb = g.decode_paged(tok, pos, layers, table, want_logits=True)
            assert np.abs(la - lb).max() <= bound, np.abs(la - lb).max()
            if kind == torch.float32:
                assert np.array_equal(a, b)
            # what a server returns beside the token: its log probability and alternatives
            r = token_logprobs(torch.from_numpy(lb).cuda(), torch.from_numpy(b.astype(np.int64)).cuda(), top=3)
            ref = log_softmax64(lb)
            assert np.abs(r.lp.cpu().numpy() - ref[np.arange(4), b]).max() < 1e-5
            top = torch.sort(torch.from_numpy(lb), dim=1, descending=True, stable=True).indices[:, :3]
            assert torch.equal(r.top_ids.cpu().long(), top)
            tok, pos = a, pos + 1


def test_decode_paged_more_sequences_than_slots_sharing_a_prefix():
    """Forty sequences over one arena slot: their common prefix lies in shared pages, the rest in their own."""
    pk = make_pack(MINI, "auto", 0, 0.02)
    eng = oracle_engine(pk)
    page, n = 8, 40
    prefix = np.arange(3, 3 + 16, dtype=np.uint32)  # two whole pages
    table = torch.full((n, 4), -1, dtype=torch.int32)
    table[:, 0], table[:, 1] = 7, 2
    table[:, 2] = torch.arange(n) + 10
    table = table.cuda()
    with Gpu(pk, max_seqs=1) as g:
        layers = caches(MINI, 60, page, torch.float32)
        g.prefill([prefix])
        g.page_out(0, prefix.size, layers, table, 0)
        tok = (np.arange(n) * 5 % MINI.vocab).astype(np.uint32)
        a, la = g.decode_paged(tok, np.full(n, 16, np.int32), layers, table, want_logits=True)
        b, lb = g.decode_paged(a, np.full(n, 17, np.int32), layers, table, want_logits=True)
        for s in (0, 13, 39):
            ref = oracle_prefix_logits(eng, np.concatenate([prefix, tok[s:s + 1], a[s:s + 1]]))
            assert np.abs(la[s] - ref[16]).max() <= observed(g) and np.abs(lb[s] - ref[17]).max() <= observed(g)


def test_paged_model_refusals():
    pk = make_pack(TINY, "auto")
    with Gpu(pk) as g:
        layers = caches(TINY, 4, 16, torch.float32)
        table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
        table[0] = torch.tensor([0, 1, 9, 2])
        g.prefill([np.arange(5, dtype=np.uint32)])
        g.page_out(0, 32, layers, table, 0)
        ok = np.array([1], np.uint32)
        for pos in ([-1], [TINY.n_ctx]):
            with pytest.raises(Gpt2qError, match="pos"):
                g.decode_paged(ok, pos, layers, table)
        with pytest.raises(Gpt2qError, match="vocab"):
            g.decode_paged([TINY.vocab], [0], layers, table)
        with pytest.raises(Gpt2qError, match="rows"):
            g.decode_paged([1, 2], [0, 0], layers, table)
        with pytest.raises(Gpt2qError, match="page"):
            g.decode_paged(ok, [32], layers, table)  # page 9 of 4
        with pytest.raises(Gpt2qError, match="page"):
            g.page_out(0, 33, layers, table, 0)
        for bad in (dict(slot=1), dict(n_tokens=0), dict(n_tokens=TINY.n_ctx + 1), dict(row=1), dict(row=-1)):
            a = dict(slot=0, n_tokens=3, row=0) | bad
            with pytest.raises(Gpt2qError):
                g.page_out(a["slot"], a["n_tokens"], layers, table, a["row"])
        with pytest.raises(ValueError):
            g.decode_paged(ok, [0], layers[:1], table)
        wrong = PagedKV(*(torch.zeros(4, 1, 16, 64, device="cuda") for _ in range(2)))
        with pytest.raises(Gpt2qError, match="heads"):
            g.decode_paged(ok, [0], [wrong, wrong], table)
        assert g.decode_paged(ok, [5], layers, table).shape == (1,)
