"""What the tests of the 8-bit paged cache and of drafted tokens share: caches of every type with their values in 64 bits, and
attention in 64 bits with a bound on the kernels' error.

The bound: u = 2^-24 is half a step of fp32. A score of D terms is within D u S, S = scale * sum |q_i k_i|; exp's argument and exp
itself add (|s| + 4) 2^-22; each of n keys adds one rounding to the sums, n u; a weight's relative error counts twice (numerator and sum).
Weights are held in 16-bit pieces: of fp16 caches and 8-bit ones 2^-20 covers two pieces, and what is under 2^-25 of the largest
weight times value scale (2^-35 of it, once for each of n keys); of bf16 caches 2^-20 covers three pieces (fp32 outputs) and 2^-16
two. A cache's q in fp32 or bf16 is exact to 2^-22 of the head's largest element in fp16 pieces, which D u S covers too as D >= 8. All of it times
the largest |v|; then the output's own rounding, e |o|. Drafted tokens' attention on wide tiles rounds each weight to one 16-bit
number: half a step, e_w = 2^-8 (bf16, 8 significant bits: spacing 2^-7 from 1 on) or 2^-11 (fp16) of itself. The product is off by e_w
of sum w |v|, the sum of the rounded weights (8-bit caches: of those before) by e_w of itself, and the logarithm by e_w."""
import math

import numpy as np
import torch

T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}
U = 2.0 ** -24
WEIGHT = (2.0 ** -11, 2.0 ** -8)  # half a step of a weight on wide tiles, of fp16 and of bf16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, kind="f32", scale=1.0):
    return torch.empty(shape, dtype=T[kind], device="cuda").normal_(0, scale, generator=g)


def quantise(x, kind):
    """(codes, scales) of fp32 entries x [..., dim], in fp32 operations."""
    x = x.float()
    top = x.abs().amax(-1)
    most = torch.full_like(top, TOP[kind])  # quotients of tensors are rounded once; those of a number and a tensor go by a reciprocal
    code = x * torch.where(top > 0, most / top, 0.0)[..., None]
    return (code.round() if kind == "i8" else code).to(T[kind]), top / most


class Cache:
    """Random pools of one cache type; `values` are what the entries stand for, in 64 bits, [2][page, head, slot, dim]."""

    def __init__(self, g, pages, heads, page, dim, kind, layout="hnd", sizes=0.5):
        from smelt_b200.paged import PagedKV

        shape = (pages, heads, page, dim) if layout == "hnd" else (pages, page, heads, dim)
        self.pools, self.scales = [], [None, None]
        for i in range(2):
            if kind in TOP:
                codes, scales = quantise(randn(g, *shape) * torch.exp(sizes * randn(g, *shape[:3], 1)), kind)
                self.scales[i] = scales if layout == "hnd" else scales.transpose(1, 2)
            else:
                codes = randn(g, *shape, kind=kind)
            self.pools.append(codes if layout == "hnd" else codes.transpose(1, 2))
        self.kind = kind
        self.kv = PagedKV(*self.pools, *self.scales)

    @property
    def values(self):
        return [p.double() if s is None else p.double() * s.double()[..., None] for p, s in zip(self.pools, self.scales)]

    def spoil(self, keep):
        """Entries [page, slot] that are not kept get NaN (of int8 codes: the scale)."""
        for p, s in zip(self.pools, self.scales):
            if s is not None:
                s.masked_fill_(~keep[:, None, :], math.nan)
                p.view(torch.int8).masked_fill_(~keep[:, None, :, None], 0x7f)
            else:
                p.masked_fill_(~keep[:, None, :, None], math.nan)

    def used(self, table, lens):
        keep = torch.zeros(self.pools[0].shape[0], self.pools[0].shape[2], dtype=torch.bool, device="cuda")
        page = keep.shape[1]
        for r, n in enumerate(lens):
            j = torch.arange(max(0, n), device="cuda")
            keep[table[r, torch.div(j, page, rounding_mode="floor")].long(), j % page] = True
        return keep


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


def attention64(q, values, table_row, keys, seen, scale):
    """(out, lse, bound before the output's rounding and the weights' pieces, largest |v|) of queries q [m, heads, dim] over the
    cached positions `keys` of one row, seen [m, keys]."""
    m, heads, dim = q.shape
    kv, page = values[0].shape[1], values[0].shape[2]
    group = heads // kv
    ids = table_row[torch.div(keys, page, rounding_mode="floor")].long()
    K, V = (x[ids, :, keys % page] for x in values)  # [keys, kv, dim]
    Q = q.double().view(m, kv, group, dim)
    hide = ~seen[:, None, None, :]
    s = (torch.einsum("mhgd,khd->mhgk", Q, K) * scale).masked_fill(hide, -math.inf)
    S = (torch.einsum("mhgd,khd->mhgk", Q.abs(), K.abs()) * abs(scale)).masked_fill(hide, 0.0)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    out = torch.einsum("mhgk,khd->mhgd", w, V)
    size = torch.einsum("mhgk,khd->mhgd", w, V.abs())  # sum w |v|
    n = len(keys)
    top = s.masked_fill(hide, 0.0).abs().amax(-1)
    rel = dim * U * S.amax(-1) + (top + 4) * 2.0 ** -22 + n * U
    vmax = V.abs().amax((0, 2))[None, :, None]
    tol = 2 * rel * vmax + n * 2.0 ** -35 * vmax
    return (out.reshape(m, heads, dim), lse.reshape(m, heads), tol.reshape(m, heads, 1), size.reshape(m, heads, dim),
            (2 * rel).reshape(m, heads), vmax.expand(m, kv, group).reshape(m, heads, 1))


def bound_of(tol, size, vmax, want, io, cache, wide=False):
    """`wide`: on tiles that round a weight to one 16-bit number."""
    e = torch.finfo(T[io]).eps / 2
    pieces = 2.0 ** -20 if io == "f32" or cache != "bf16" else 2.0 ** -16
    t = tol + pieces * vmax + want.abs() * e * 1.01 + (2.0 ** -25 if io == "f16" else 0)
    if wide and io != "f32":
        t = t + 2 * WEIGHT[cache == "bf16"] * size
    return t


def close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    over = float((err - tol).max()) if err.numel() else 0.0
    assert over <= 0, (what, over, float(err.max()))
