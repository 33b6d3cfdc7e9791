"""A paged key/value cache on the device: appending tokens, reading them back, and attention of one new token or of
a tree of drafted tokens per row.

    kv = PagedKV(k_pool, v_pool)                 # [pages, kv heads, page size, head dim]
    kv = PagedKV(k_codes, v_codes, k_scale, v_scale)   # int8 or float8_e4m3fn, a scale per entry
    rotary = Rotary(head_dim)
    q = kv.append(k, v, table, pos, seq=seq, rotary=rotary, q=q)
    out = kv.attend(q, table, lens)

A step with drafted tokens, of which `accept` is decided from its results:

    mask, depth = tree_mask(parents)             # one list of parents per row
    q = kv.append(k, v, table, lens[seq] + depth, seq=seq, rotary=rotary, q=q, slot=lens[seq] + node)
    out = kv.attend_tree(q, table, lens, first, mask)
    lens = kv.commit(table, lens, accept)

The tensors are torch CUDA tensors; calls go to the current torch stream and may be captured into a
CUDA graph. include/gpt2q.h (gpt2q_paged_*) states the layout and what each call does with padding,
empty rows and bad page ids.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _ffi
from .device import CODES, DTYPES, ops

STATUS_PAGE, STATUS_POSITION, STATUS_ROW, STATUS_TIMEOUT = 1, 2, 4, 8


class Rotary:
    """Position rotation of the first `dim` elements of a head: pair i is turned by
    position * base^(-2i/dim) radians, or by position * inv_freq[i] when those are given. Pairs are
    (i, i + dim/2), or (2i, 2i + 1) with interleaved=True."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, inv_freq=None):
        lib = _ffi.load()
        self.c = _ffi.Rotary()
        _ffi.check(lib, None, lib.gpt2q_rotary_init(C.byref(self.c), int(dim), 1 if interleaved else 0, float(base)))
        if inv_freq is not None:
            f = [float(x) for x in inv_freq]
            if len(f) != dim // 2 or not all(math.isfinite(x) for x in f):
                raise ValueError(f"inv_freq must have {dim // 2} finite elements")
            for i, x in enumerate(f):
                self.c.turns[i] = x / (2.0 * math.pi)
        self.address = C.addressof(self.c)

    def __setstate__(self, state):
        """Of a copy or an unpickled object: the address of its own structure."""
        self.__dict__.update(state)
        self.address = C.addressof(self.c)


class PagedKV:
    """One layer's cache over two pools of pages [n_pages, n_kv_heads, page_size, head_dim], which
    the caller keeps: any strides that both share, multiples of 16 bytes, unit stride over the head
    dim ([n_pages, page_size, n_kv_heads, head_dim] storage is its transposed view).

    Pools of int8 or float8_e4m3fn hold codes: an entry (one token's head_dim elements of a head) stands for code *
    scale, with k_scale and v_scale [n_pages, n_kv_heads, page_size] float32 of any strides that both share, and
    head_dim a multiple of 16. append() sets both; the other tensors of calls may be float32, float16 or bfloat16."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        if not (k.is_cuda and v.is_cuda and k.get_device() == v.get_device()):
            raise ValueError("the pools must be on one CUDA device")
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("the pools must be [pages, kv heads, page size, head dim]")
        eight = k.dtype in CODES
        if not (eight or k.dtype in DTYPES) or v.dtype != k.dtype:
            raise ValueError("the pools must be float32, float16, bfloat16, int8 or float8_e4m3fn")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("the pools must share their strides, unit over the head dim")
        if (k_scale is None) != (v_scale is None) or eight != (k_scale is not None):
            raise ValueError("pools of 8 bits come with k_scale and v_scale, others without")
        ffi = ops()
        self._append, self._attend, self._attend_tree, self._read, self._commit = (
            ffi.append, ffi.attend, ffi.attend_tree, ffi.read, ffi.commit)
        self._pools = k, v, k_scale, v_scale  # `c` holds their addresses
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.index = k.dtype, k.get_device()
        self.c = _ffi.PagedKV(k.data_ptr(), v.data_ptr(), CODES[k.dtype] if eight else DTYPES[k.dtype],
                              *(k.shape[i] for i in (0, 2, 1, 3)), _ffi.SCALED if eight else 0,
                              k.stride(0), k.stride(1), k.stride(2))
        if eight:
            for s in (k_scale, v_scale):
                if not s.is_cuda or s.get_device() != self.index or s.dtype != torch.float32 or s.shape != k.shape[:3]:
                    raise ValueError("the scales must be float32 [pages, kv heads, page size] on the pools' device")
            if k_scale.stride() != v_scale.stride():
                raise ValueError("the scales must share their strides")
            self.c = _ffi.PagedKV8(self.c, k_scale.data_ptr(), v_scale.data_ptr(), *k_scale.stride())
        self.address = C.addressof(self.c)

    @property
    def k(self):
        return self._pools[0]

    @property
    def v(self):
        return self._pools[1]

    @property
    def k_scale(self):
        return self._pools[2]

    @property
    def v_scale(self):
        return self._pools[3]

    def append(self, k, v, table, pos, seq=None, rotary: Rotary | None = None, q=None, q_out=None, status=None, slot=None):
        """Writes token i's k[i] and v[i] ([tokens, kv heads, head dim]) at position pos[i] of table row
        seq[i] (seq None: row i), keys rotated by `rotary`. With q ([tokens, heads, head dim]) the queries
        are rotated too, into q_out (a new tensor when None; q itself may be given), which is returned.
        pos[i] < 0 marks padding. With `slot` the entry goes to position slot[i] of the row and pos[i] is only the
        rotation's. `status` is an int32 tensor of one element that collects STATUS_* bits."""
        return self._append(self.address, self.index, k, v, table, pos, seq, None if rotary is None else rotary.address,
                            q, q_out, status, slot)

    def read(self, table, pos, seq=None, dtype=None, k=None, v=None, status=None):
        """(k, v), [tokens, kv heads, head dim] each: the cached entries of position pos[i] of table row seq[i] (seq None:
        row i), zeros for pos[i] < 0. `dtype` is that of new tensors: the cache's (bfloat16 for 8 bits) unless given."""
        if dtype is None:
            dtype = torch.bfloat16 if self.dtype in CODES else self.dtype
        if dtype not in DTYPES or (self.dtype not in CODES and dtype not in (self.dtype, torch.float32)):
            raise ValueError("dtype must be the cache's or float32, of an 8-bit cache float32, float16 or bfloat16")
        return self._read(self.address, self.index, table, pos, seq, k, v, DTYPES[dtype], status)

    def attend(self, q, table, lens, scale: float | None = None, window: int = 0, out=None, lse=None, status=None):
        """Attention of one query per table row ([rows, heads, head dim]) over the last `window` (0: all) of
        the row's first lens[row] cached tokens; scale defaults to 1/sqrt(head dim). Returns out. `lse`
        ([rows, heads] float32, contiguous) receives the log of each sum of exp."""
        return self._attend(self.address, self.index, q, table, lens, scale, window, out, lse, status)

    def attend_tree(self, q, table, lens, first, mask=None, scale: float | None = None, out=None, lse=None, status=None):
        """Attention of drafted tokens, [tokens, heads, head dim]: row r has tokens first[r] .. first[r + 1] - 1 (`first`
        [rows + 1] int32), which are cached behind the row's lens[r] tokens. Each sees those and, of its row's drafted
        tokens, the ones its mask names: bit j & 31 of mask[token, j // 32] (int32, see tree_mask); None: itself and
        those before it. Returns out; `lse` is [tokens, heads]. Tokens of no row are left as they were."""
        return self._attend_tree(self.address, self.index, q, table, lens, scale, first, mask, out, lse, status)

    def commit(self, table, lens, accept, new_lens=None, status=None):
        """Moves the accepted drafted tokens behind their rows: entry lens[r] + accept[r, i] goes to position lens[r] + i;
        accept [rows, tokens] int32 rises along a row, and a negative element ends it. Returns the new lengths."""
        return self._commit(self.address, self.index, table, lens, accept, new_lens, status)


def tree_mask(parents, device="cuda"):
    """(mask, depth) of drafted trees for attend_tree and append: `parents` is one list per row, the parent of each of its
    tokens among the row's earlier ones, or -1 for one that follows the row's last token. mask [tokens, words] int32 names
    a token's ancestors and itself, depth [tokens] int32 counts the ancestors. Made on the host."""
    seen, depth, most = [], [], 1
    for row in parents:
        at = len(seen)
        most = max(most, len(row))
        for i, p in enumerate(row):
            p = int(p)
            if not -1 <= p < i:
                raise ValueError("a token's parent must be an earlier token of its row, or -1")
            seen.append((seen[at + p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[at + p] + 1 if p >= 0 else 0)
    words = (most + 31) // 32
    raw = b"".join(m.to_bytes(4 * words, "little") for m in seen)
    mask = torch.frombuffer(bytearray(raw), dtype=torch.int32) if raw else torch.empty(0, dtype=torch.int32)
    return mask.view(-1, words).to(device), torch.tensor(depth, dtype=torch.int32).to(device)
