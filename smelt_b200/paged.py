"""A paged key/value cache on the device: appending tokens, and attention of one new token per row.

    kv = PagedKV(k_pool, v_pool)                 # [pages, kv heads, page size, head dim]
    rotary = Rotary(head_dim)
    q = kv.append(k, v, table, pos, seq=seq, rotary=rotary, q=q)
    out = kv.attend(q, table, lens)

The tensors are torch CUDA tensors; calls go to the current torch stream and may be captured into a
CUDA graph. include/gpt2q.h (gpt2q_paged_*) states the layout and what each call does with padding,
empty rows and bad page ids.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _ffi
from .device import DTYPES, call, ints, need, on_device

STATUS_PAGE, STATUS_POSITION, STATUS_ROW = 1, 2, 4


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
            need(len(f) == dim // 2, f"inv_freq must have {dim // 2} elements")
            for i, x in enumerate(f):
                need(math.isfinite(x), "inv_freq must be finite")
                self.c.turns[i] = x / (2.0 * math.pi)
        self.ref = C.byref(self.c)


def _heads(t, index: int, name: str, n: int, heads: int, dim: int, dtype):
    on_device(t, index, name)
    if t.shape != (n, heads, dim) or t.dtype != dtype:
        raise ValueError(f"{name} must be [{n}, {heads}, {dim}] of {dtype}")
    st, sh, sd = t.stride()
    if sd != 1 and dim > 1:
        raise ValueError(f"{name} must have unit stride over the head dim")
    return _ffi.Heads(t.data_ptr(), st, sh)


class PagedKV:
    """One layer's cache over two pools of pages [n_pages, n_kv_heads, page_size, head_dim], which
    the caller keeps: any strides that both share, multiples of 16 bytes, unit stride over the head
    dim ([n_pages, page_size, n_kv_heads, head_dim] storage is its transposed view)."""

    def __init__(self, k, v):
        need(k.is_cuda and v.is_cuda and k.get_device() == v.get_device(), "the pools must be on one CUDA device")
        need(k.dim() == 4 and k.shape == v.shape, "the pools must be [pages, kv heads, page size, head dim]")
        need(k.dtype in DTYPES and v.dtype == k.dtype, "the pools must be float32, float16 or bfloat16")
        need(k.stride() == v.stride() and k.stride(3) == 1, "the pools must share their strides, unit over the head dim")
        self._lib = _ffi.load()
        self.k, self.v = k, v
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.index = k.dtype, k.get_device()
        self.c = _ffi.PagedKV(k.data_ptr(), v.data_ptr(), DTYPES[k.dtype], *(k.shape[i] for i in (0, 2, 1, 3)), 0,
                              k.stride(0), k.stride(1), k.stride(2))
        self.ref = C.byref(self.c)
        self._work = {}  # heads -> workspace bytes

    def _type(self, t):
        if t.dtype != self.dtype and t.dtype != torch.float32:
            raise ValueError(f"tensors must be {self.dtype} like the cache, or float32")
        return t.dtype

    def _table(self, table):
        on_device(table, self.index, "table")
        if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("table must be int32 [rows, pages] with unit stride over the pages")
        rows, width = table.shape
        return _ffi.PageTable(table.data_ptr(), rows, width, max(table.stride(0), width))

    def append(self, k, v, table, pos, seq=None, rotary: Rotary | None = None, q=None, q_out=None, status=None):
        """Writes token i's k[i] and v[i] ([tokens, kv heads, head dim]) at position pos[i] of table row
        seq[i] (seq None: row i), keys rotated by `rotary`. With q ([tokens, heads, head dim]) the queries
        are rotated too, into q_out (a new tensor when None; q itself may be given), which is returned.
        pos[i] < 0 marks padding. `status` is an int32 tensor of one element that collects STATUS_* bits."""
        n, dtype = k.shape[0], self._type(k)
        kh = _heads(k, self.index, "k", n, self.n_kv_heads, self.head_dim, dtype)
        vh = _heads(v, self.index, "v", n, self.n_kv_heads, self.head_dim, dtype)
        ints(pos, self.index, "pos", n)
        if seq is not None:
            ints(seq, self.index, "seq", n)
        if status is not None:
            ints(status, self.index, "status", 1)
        qh = oh = None
        heads = 0
        if q is not None:
            heads = q.shape[1]
            qh = C.byref(_heads(q, self.index, "q", n, heads, self.head_dim, dtype))
            if q_out is None:
                q_out = torch.empty((n, heads, self.head_dim), dtype=dtype, device=q.device)
            oh = C.byref(_heads(q_out, self.index, "q_out", n, heads, self.head_dim, dtype))
        elif q_out is not None:
            raise ValueError("q_out without q")
        call(self._lib.gpt2q_paged_append, self.index, self.ref, C.byref(self._table(table)), C.byref(kh), C.byref(vh),
             qh, oh, DTYPES[dtype], heads, n, pos.data_ptr(), None if seq is None else seq.data_ptr(),
             None if rotary is None else rotary.ref, None if status is None else status.data_ptr())
        return q_out

    def attend(self, q, table, lens, scale: float | None = None, window: int = 0, out=None, lse=None, status=None):
        """Attention of one query per table row ([rows, heads, head dim]) over the last `window` (0: all) of
        the row's first lens[row] cached tokens; scale defaults to 1/sqrt(head dim). Returns out. `lse`
        ([rows, heads] float32, contiguous) receives the log of each sum of exp."""
        dtype = self._type(q)
        n, heads, _ = q.shape
        qh = _heads(q, self.index, "q", n, heads, self.head_dim, dtype)
        ints(lens, self.index, "lens", n)
        t = self._table(table)
        if t.n_rows != n:
            raise ValueError(f"table must have {n} rows")
        if out is None:
            out = torch.empty((n, heads, self.head_dim), dtype=dtype, device=q.device)
        oh = _heads(out, self.index, "out", n, heads, self.head_dim, dtype)
        if lse is not None:
            on_device(lse, self.index, "lse")
            need(lse.dtype == torch.float32 and lse.shape == (n, heads) and lse.is_contiguous(),
                 f"lse must be a contiguous float32 tensor [{n}, {heads}]")
        if status is not None:
            ints(status, self.index, "status", 1)
        size = self._work.get(heads)
        if size is None:
            size = self._work[heads] = int(self._lib.gpt2q_paged_attention_workspace(self.ref, heads))
        # from torch's allocator on every call: calls on other streams and captured graphs each get their own
        work = torch.empty(max(16, size), dtype=torch.uint8, device=q.device)
        call(self._lib.gpt2q_paged_attention, self.index, self.ref, C.byref(t), lens.data_ptr(), C.byref(qh),
             C.byref(oh), DTYPES[dtype], heads, self.head_dim ** -0.5 if scale is None else scale, window,
             None if lse is None else lse.data_ptr(), None if status is None else status.data_ptr(), work.data_ptr())
        return out
