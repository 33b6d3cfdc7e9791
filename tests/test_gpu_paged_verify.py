"""Drafted tokens and 8-bit caches through the model (gpt2q_verify_paged, gpt2q_commit_paged, gpt2q_page_out and
gpt2q_decode_paged over gpt2q_paged_kv8).

Tolerances: fp32 caches within the handle's own bound of the oracle's logits. A cache that rounds keys and values moves the
logits in proportion to its half step: fp16 (2^-12 of the value) is accepted at 2e-2, so int8 (an entry's largest / 254, at most 2^-7.9 of a
value's bound) at 2e-2 * 2^4.1 and e4m3 (2^-4) at 2e-2 * 2^8."""
import numpy as np
import pytest
import torch

from smelt_b200._ffi import Gpt2qError
from smelt_b200.gpu import Gpu
from smelt_b200.paged import PagedKV

from .helpers import MINI, TINY, make_pack, observed, oracle_engine, oracle_prefix_logits

pytestmark = pytest.mark.gpu
KINDS = [(torch.float32, None), (torch.float16, 2e-2), (torch.int8, 2e-2 * 2 ** 4.1), (torch.float8_e4m3fn, 2e-2 * 2 ** 8)]


@pytest.fixture(scope="module", autouse=True)
def _built():
    from smelt_b200 import build
    build.build()


def caches(meta, pages, page, kind):
    hd = meta.n_embd // meta.n_head
    out = []
    for _ in range(meta.n_layer):
        if kind.itemsize == 1:
            k, v = (torch.full((pages, page, meta.n_head, hd), 0x7f, dtype=torch.int8, device="cuda").view(kind).transpose(1, 2) for _ in range(2))
            out.append(PagedKV(k, v, *(torch.full((pages, meta.n_head, page), float("nan"), device="cuda") for _ in range(2))))
        else:
            k, v = (torch.full((pages, page, meta.n_head, hd), float("nan"), dtype=kind, device="cuda").transpose(1, 2) for _ in range(2))
            out.append(PagedKV(k, v))
    return out


def path_to(parents, node):
    path = []
    while node >= 0:
        path.append(node)
        node = parents[node]
    return path[::-1]


@pytest.mark.parametrize("kind,bound", KINDS)
@pytest.mark.parametrize("meta,policy,page", [(MINI, "auto", 16), (MINI, "f32", 5), (TINY, "q4auto", 64)])
def test_verified_trees_match_the_oracle_and_decode(kind, bound, meta, policy, page):
    pk = make_pack(meta, policy, 0, 0.02)
    eng = oracle_engine(pk)
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, meta.vocab, n).astype(np.uint32) for n in (5, 1, 17, 9)]
    width = -(-meta.n_ctx // page)
    table = torch.from_numpy(rng.permutation(4 * width).astype(np.int32).reshape(4, width)).cuda()
    with Gpu(pk, max_seqs=4, max_tokens=128) as g:
        e = observed(g) if bound is None else bound
        a, b = caches(meta, 4 * width, page, kind), caches(meta, 4 * width, page, kind)
        g.prefill(prompts)
        for s, p in enumerate(prompts):
            g.page_out(s, p.size, a, table, s)
            g.page_out(s, p.size, b, table, s)
        text = [list(p) for p in prompts]
        lens = np.array([p.size for p in prompts], np.int32)
        for step in range(2):
            sizes = [(9, 1, 0, 6), (3, 8, 33, 1)][step]
            parents = [[-1] + [int(rng.integers(max(-1, i - 4), i)) for i in range(1, n)] if n else [] for n in sizes]
            depth = [max((len(path_to(p, i)) for i in range(len(p))), default=0) for p in parents]
            assert all(n + d <= meta.n_ctx for n, d in zip(lens, depth))
            drafts = [rng.integers(0, meta.vocab, n).astype(np.uint32) for n in sizes]
            nxt, lg = g.verify_paged(drafts, parents, lens, a, table, want_logits=True)
            assert [len(x) for x in nxt] == list(sizes) and [x.shape for x in lg] == [(n, meta.vocab) for n in sizes]
            accept = []
            for s in range(4):
                for i in range(sizes[s]):
                    path = path_to(parents[s], i)
                    if i in (0, sizes[s] // 2, sizes[s] - 1):
                        ref = oracle_prefix_logits(eng, np.array(text[s] + [drafts[s][j] for j in path], np.uint32))[-1]
                        assert np.abs(lg[s][i] - ref).max() <= e, (s, i, np.abs(lg[s][i] - ref).max())
                    assert nxt[s][i] == lg[s][i].argmax()
                accept.append(path_to(parents[s], int(rng.integers(0, sizes[s]))) if sizes[s] else [])
            # the accepted tokens one by one over the other caches
            for i in range(max(map(len, accept))):
                rows = [s for s in range(4) if i < len(accept[s])]
                one, lo = g.decode_paged([drafts[s][accept[s][i]] for s in rows], [lens[s] + i for s in rows], b, table[rows].contiguous(), want_logits=True)
                for s, l in zip(rows, lo):
                    assert np.abs(lg[s][accept[s][i]] - l).max() <= 2 * e
            new = g.commit_paged(lens, accept, a, table)
            assert new.tolist() == [n + len(x) for n, x in zip(lens, accept)]
            for s in range(4):
                text[s] += [drafts[s][j] for j in accept[s]]
            lens = new
            # what both hold: the tokens' keys and values up to the arithmetic's difference, in the same places
            for x, y in zip(a, b):
                for s in range(4):
                    at = torch.arange(int(lens[s]), dtype=torch.int32, device="cuda")
                    row = torch.full_like(at, s)
                    for u, w in zip(x.read(table, at, seq=row, dtype=torch.float32), y.read(table, at, seq=row, dtype=torch.float32)):
                        step_of = {torch.float32: 1e-3, torch.float16: 2.0 ** -9, torch.int8: 1 / 60, torch.float8_e4m3fn: 2.0 ** -2}[kind]
                        assert bool(((u - w).abs() <= step_of * u.abs().amax(-1, keepdim=True) + 1e-3).all())
        tok = [int(t[-1]) for t in text]
        a2, la = g.decode_paged(tok, lens, a, table, want_logits=True)
        b2, lb = g.decode_paged(tok, lens, b, table, want_logits=True)
        assert np.abs(la - lb).max() <= 2 * e


def test_speculative_greedy_equals_greedy():
    """Drafts are guesses (some of them right); whatever is accepted, the text is that of greedy decoding."""
    pk = make_pack(MINI, "auto", 0, 0.02)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, MINI.vocab, n).astype(np.uint32) for n in (7, 3)]
    page = 8
    width = -(-MINI.n_ctx // page)
    table = torch.arange(2 * width, dtype=torch.int32, device="cuda").view(2, width)
    steps = 20
    with Gpu(pk, max_seqs=2, max_tokens=64) as g:
        want = g.generate_greedy(prompts, steps + 8)
        layers = caches(MINI, 2 * width, page, torch.float32)
        first = g.prefill(prompts)
        for s, p in enumerate(prompts):
            g.page_out(s, p.size, layers, table, s)
        got = [[int(t)] for t in first]
        lens = np.array([p.size for p in prompts], np.int32)
        kept = 0
        while min(map(len, got)) < steps:
            drafts, parents = [], []
            for s in range(2):
                at = len(got[s])
                right = [int(want[s][min(at + i, steps + 7)]) for i in range(3)]
                wrong = rng.integers(0, MINI.vocab, 4).tolist()
                # the last token, then two branches of which one begins as the model would go on
                drafts.append(np.array([got[s][-1], wrong[0], right[0], wrong[1], right[1], wrong[2], right[2]], np.uint32))
                parents.append([-1, 0, 0, 1, 2, 4, 4])
            nxt = g.verify_paged(drafts, parents, lens, layers, table)
            accept = []
            for s in range(2):
                path, go = [0], True
                while go:
                    pick = int(nxt[s][path[-1]])
                    got[s].append(pick)
                    more = [i for i in range(path[-1] + 1, 7) if parents[s][i] == path[-1] and int(drafts[s][i]) == pick]
                    go = bool(more)
                    path += more[:1]
                accept.append(path)
                kept += len(path) - 1
            lens = g.commit_paged(lens, accept, layers, table)
        assert kept > 4
        for s in range(2):
            assert got[s][:steps] == [int(t) for t in want[s][:steps]]


@pytest.mark.parametrize("kind,bound", KINDS[2:])
def test_decode_over_8_bit_caches(kind, bound):
    pk = make_pack(MINI, "auto", 0, 0.02)
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, MINI.vocab, n).astype(np.uint32) for n in (5, 1, 40, 17)]
    width = -(-MINI.n_ctx // 16)
    table = torch.from_numpy(rng.permutation(4 * width).astype(np.int32).reshape(4, width)).cuda()
    with Gpu(pk, max_seqs=4) as g:
        layers = caches(MINI, 4 * width, 16, kind)
        tok = g.prefill(prompts)
        for s, p in enumerate(prompts):
            g.page_out(s, p.size, layers, table, s)
        pos = np.array([p.size for p in prompts], np.int32)
        for _ in range(6):
            a, la = g.decode(tok, pos, want_logits=True)
            _, lb = g.decode_paged(tok, pos, layers, table, want_logits=True)
            assert 0 < np.abs(la - lb).max() <= bound
            tok, pos = a, pos + 1


def test_refusals():
    pk = make_pack(TINY, "auto")
    with Gpu(pk, max_tokens=16) as g:
        layers = caches(TINY, 8, 16, torch.float32)
        table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
        ok = dict(drafts=[np.array([1, 2], np.uint32), np.array([3], np.uint32)], parents=[[-1, 0], [-1]], lens=[0, 0])
        assert [len(x) for x in g.verify_paged(**ok, layers=layers, table=table)] == [2, 1]
        for bad, text in ((dict(parents=[[-1, 1], [-1]]), "parent"), (dict(parents=[[-2, 0], [-1]]), "parent"), (dict(lens=[0, -1]), "lens"),
                          (dict(lens=[TINY.n_ctx - 1, 0]), "n_ctx"), (dict(drafts=[np.array([1, TINY.vocab], np.uint32), np.array([3], np.uint32)]), "vocab"),
                          (dict(drafts=[np.zeros(0, np.uint32)] * 2, parents=[[], []]), "drafted"),
                          (dict(drafts=[np.zeros(400, np.uint32), np.zeros(1, np.uint32)], parents=[[-1] * 400, [-1]]), "drafted")):
            with pytest.raises(Gpt2qError, match=text):
                g.verify_paged(**(ok | bad), layers=layers, table=table)
        with pytest.raises(ValueError):
            g.verify_paged(**(ok | dict(parents=[[-1], [-1]])), layers=layers, table=table)
        with pytest.raises(ValueError):
            g.verify_paged(**(ok | dict(lens=[0])), layers=layers, table=table)
        with pytest.raises(Gpt2qError, match="rows"):
            g.verify_paged(**ok, layers=layers, table=table[:1])
        with pytest.raises(ValueError):
            g.commit_paged([0, 0], [[0]], layers, table)
        far = torch.full((2, 4), 99, dtype=torch.int32, device="cuda")
        with pytest.raises(Gpt2qError, match="page"):
            g.verify_paged(**ok, layers=layers, table=far)
        with pytest.raises(Gpt2qError, match="page"):
            g.commit_paged([0, 0], [[1], []], layers, far)
        mixed = [layers[0], *caches(TINY, 8, 16, torch.int8)[1:]]
        with pytest.raises(ValueError, match="8 bits"):
            g.verify_paged(**ok, layers=mixed, table=table)
        assert g.commit_paged([1, 0], [[1], [0]], layers, table).tolist() == [2, 1]
