"""The model over 8-bit paged caches against a forward in 64 bits whose keys and values are quantised as the cache's are.

The prompt's own forward has exact keys and values (the arena's), which are quantised when they are paged out; tokens behind it
attend over quantised ones, their own included.

Tolerance: let N be how far quantising moves a token's logits (largest difference of the two forwards). The handle's keys are off by some
1e-6 of their entry's largest element before they are quantised, so that a part in a thousand of the codes (127 steps of
int8; e4m3's are wider) come out one step away, where a code is off by up to half a step anyway: a variance of 1e-3 steps against 1/12, a
ninth of N. N / 2 and the handle's own accuracy leave room for later layers, and what is wrong moves the logits by more than 3 N
(test_a_wrong_tree_is_noticed)."""
import numpy as np
import pytest
import torch

from oracle import backward_oracle as B
from smelt_b200.gpu import Gpu
from smelt_b200.paged import PagedKV

from .helpers import MINI, make_pack, observed

KINDS = {"i8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def held(x, kind, heads):
    """What the cache holds of entries x [tokens, heads * dim]."""
    t = torch.from_numpy(x.astype(np.float32)).view(len(x), heads, -1)
    top = t.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, KINDS[kind][1])
    code = t * torch.where(top > 0, most / top, 0.0)
    code = code.round() if kind == "i8" else code.to(torch.float8_e4m3fn).float()
    return (code.double() * (top / most).double()).reshape(len(x), -1).numpy()


def forward(W, meta, ids, pos, sees, prompt, kind):
    """Logits of every token; sees[i, j]: token i attends over token j. Tokens from `prompt` on attend over the cache of type `kind`."""
    E, H = meta.n_embd, meta.n_head
    hd = E // H
    x = W["wte.weight"][ids] + W["wpe.weight"][pos]
    for l in range(meta.n_layer):
        p = f"h.{l}."
        h = B.layernorm(x, W[p + "ln_1.weight"], W[p + "ln_1.bias"], meta.ln_eps)
        qkv = h @ W[p + "attn.c_attn.weight"].T + W[p + "attn.c_attn.bias"]
        q, k, v = qkv[:, :E], qkv[:, E:2 * E], qkv[:, 2 * E:]
        o = np.zeros_like(q)
        for rows, kk, vv in ((slice(0, prompt), k, v), (slice(prompt, None), held(k, kind, H) if kind else k, held(v, kind, H) if kind else v)):
            for a in range(H):
                c = slice(a * hd, (a + 1) * hd)
                s = np.where(sees[rows], (q[rows, c] @ kk[:, c].T) / np.sqrt(hd), -np.inf)
                if len(s):
                    s = np.exp(s - s.max(1, keepdims=True))
                    o[rows, c] = (s / s.sum(1, keepdims=True)) @ vv[:, c]
        x = x + o @ W[p + "attn.c_proj.weight"].T + W[p + "attn.c_proj.bias"]
        h = B.layernorm(x, W[p + "ln_2.weight"], W[p + "ln_2.bias"], meta.ln_eps)
        x = x + B.gelu(h @ W[p + "mlp.c_fc.weight"].T + W[p + "mlp.c_fc.bias"]) @ W[p + "mlp.c_proj.weight"].T + W[p + "mlp.c_proj.bias"]
    return B.layernorm(x, W["ln_f.weight"], W["ln_f.bias"], meta.ln_eps) @ W["wte.weight"].T


def tree_of(rng, prompt, n):
    """Parents, positions and who sees whom of n drafted tokens behind a prompt."""
    parents = [-1 if i == 0 or rng.random() < 0.1 else int(rng.integers(max(-1, i - 4), i)) for i in range(n)]
    sees = np.tril(np.ones((prompt + n, prompt + n), bool))
    pos = np.arange(prompt + n)
    for i, p in enumerate(parents):
        row = np.zeros(prompt + n, bool)
        row[:prompt] = True
        if p >= 0:
            row |= sees[prompt + p]
        row[prompt + i] = True
        sees[prompt + i] = row
        pos[prompt + i] = prompt if p < 0 else pos[prompt + p] + 1
    return parents, pos, sees


CASES = [(21, 30), (5, 9), (90, 40)]


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("prompt,n", CASES)
def test_a_wrong_tree_is_noticed(kind, prompt, n):
    """A parent that is not seen, a token's position one on, or the prompt's last token not seen: further from the right logits than
    twice the tolerance (of a handle good to 1e-3)."""
    pk = make_pack(MINI, "auto", 0, 0.02)
    W, rng = B.weights64(pk), np.random.default_rng(5)
    parents, pos, sees = tree_of(rng, prompt, n)
    ids = rng.integers(0, MINI.vocab, prompt + n)
    right = forward(W, MINI, ids, pos, sees, prompt, kind)
    N = np.abs(right - forward(W, MINI, ids, pos, sees, prompt, None)).max(1)
    at = prompt + n - 1
    while parents[at - prompt] < 0:
        at -= 1
    for what in ("parent", "position", "prompt"):
        s, p = sees.copy(), pos.copy()
        if what == "parent":
            s[at, prompt + parents[at - prompt]] = False
        elif what == "prompt":
            s[at, prompt - 1] = False
        else:
            p[at] += 1
        wrong = np.abs(forward(W, MINI, ids, p, s, prompt, kind)[at] - right[at]).max()
        assert wrong > 2 * (N[at] / 2 + 1e-3), (what, wrong, N[at])


def caches(meta, pages, page, kind):
    hd = meta.n_embd // meta.n_head
    out = []
    for _ in range(meta.n_layer):
        k, v = (torch.full((pages, meta.n_head, page, hd), 0x7f, dtype=torch.int8, device="cuda").view(KINDS[kind][0]) for _ in range(2))
        out.append(PagedKV(k, v, *(torch.full((pages, meta.n_head, page), float("nan"), device="cuda") for _ in range(2))))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_trees_and_steps_over_8_bit_caches(kind):
    """Two sequences at a time: a tree of drafted tokens, its last path committed, then single tokens behind it."""
    from smelt_b200 import build
    build.build()
    pk = make_pack(MINI, "auto", 0, 0.02)
    W, rng, page = B.weights64(pk), np.random.default_rng(6), 16
    width = -(-(MINI.n_ctx + 40) // page)
    table = torch.from_numpy(rng.permutation(2 * width).astype(np.int32).reshape(2, width)).cuda()
    with Gpu(pk, max_seqs=2, max_tokens=256) as g:
        own = observed(g)
        for (p0, n0), (p1, n1) in ((CASES[0], CASES[1]), (CASES[2], CASES[0])):
            layers = caches(MINI, 2 * width, page, kind)
            shapes = [(p0, n0), (p1, n1)]
            trees = [tree_of(rng, p, n) for p, n in shapes]
            ids = [rng.integers(0, MINI.vocab, p + n) for p, n in shapes]
            g.prefill([i[:p].astype(np.uint32) for i, (p, _) in zip(ids, shapes)])
            for s, (p, _) in enumerate(shapes):
                g.page_out(s, p, layers, table, s)
            lens = np.array([p0, p1], np.int32)
            _, lg = g.verify_paged([i[p:].astype(np.uint32) for i, (p, _) in zip(ids, shapes)], [t[0] for t in trees], lens, layers, table, want_logits=True)
            paths = []
            for s, ((p, n), (parents, pos, sees)) in enumerate(zip(shapes, trees)):
                want = forward(W, MINI, ids[s], pos, sees, p, kind)[p:]
                N = np.abs(want - forward(W, MINI, ids[s], pos, sees, p, None)[p:]).max(1)
                err = np.abs(lg[s] - want).max(1)
                assert (err <= N / 2 + own).all(), (s, float((err / N).max()), float(err.max()))
                path, at = [], n - 1
                while at >= 0:
                    path, at = [at, *path], parents[at]
                paths.append(path)
            lens = g.commit_paged(lens, paths, layers, table)
            text = [np.concatenate([ids[s][:p], ids[s][p:][paths[s]]]) for s, (p, _) in enumerate(shapes)]
            for _ in range(3):
                tok = rng.integers(0, MINI.vocab, 2)
                _, lo = g.decode_paged(tok.astype(np.uint32), lens, layers, table, want_logits=True)
                text = [np.append(t, k) for t, k in zip(text, tok)]
                lens = lens + 1
                for s, (p, _) in enumerate(shapes):
                    m = len(text[s])
                    chain = np.tril(np.ones((m, m), bool))
                    want = forward(W, MINI, text[s], np.arange(m), chain, p, kind)[-1]
                    N = np.abs(want - forward(W, MINI, text[s], np.arange(m), chain, p, None)[-1]).max()
                    err = np.abs(lo[s] - want).max()
                    assert err <= N / 2 + own, (s, err / N, err)
