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

from . import _ffi
from .device import DTYPES, ops

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
    dim ([n_pages, page_size, n_kv_heads, head_dim] storage is its transposed view)."""

    def __init__(self, k, v):
        if not (k.is_cuda and v.is_cuda and k.get_device() == v.get_device()):
            raise ValueError("the pools must be on one CUDA device")
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError("the pools must be [pages, kv heads, page size, head dim]")
        if k.dtype not in DTYPES or v.dtype != k.dtype:
            raise ValueError("the pools must be float32, float16 or bfloat16")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("the pools must share their strides, unit over the head dim")
        self._append, self._attend = ops().append, ops().attend
        self._pools = k, v  # `c` holds their addresses
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.index = k.dtype, k.get_device()
        self.c = _ffi.PagedKV(k.data_ptr(), v.data_ptr(), DTYPES[k.dtype], *(k.shape[i] for i in (0, 2, 1, 3)), 0,
                              k.stride(0), k.stride(1), k.stride(2))
        self.address = C.addressof(self.c)

    @property
    def k(self):
        return self._pools[0]

    @property
    def v(self):
        return self._pools[1]

    def append(self, k, v, table, pos, seq=None, rotary: Rotary | None = None, q=None, q_out=None, status=None):
        """Writes token i's k[i] and v[i] ([tokens, kv heads, head dim]) at position pos[i] of table row
        seq[i] (seq None: row i), keys rotated by `rotary`. With q ([tokens, heads, head dim]) the queries
        are rotated too, into q_out (a new tensor when None; q itself may be given), which is returned.
        pos[i] < 0 marks padding. `status` is an int32 tensor of one element that collects STATUS_* bits."""
        return self._append(self.address, self.index, k, v, table, pos, seq, None if rotary is None else rotary.address,
                            q, q_out, status)

    def attend(self, q, table, lens, scale: float | None = None, window: int = 0, out=None, lse=None, status=None):
        """Attention of one query per table row ([rows, heads, head dim]) over the last `window` (0: all) of
        the row's first lens[row] cached tokens; scale defaults to 1/sqrt(head dim). Returns out. `lse`
        ([rows, heads] float32, contiguous) receives the log of each sum of exp."""
        return self._attend(self.address, self.index, q, table, lens, scale, window, out, lse, status)
