"""Python mirror of model-lab's CUDA executor API on top of libgpt2q.so.

`Gpu` keeps the shape of LukasParke/smelt's `Gpu` (experiments/model-lab/src/
gpu.rs:51-379): construct from a weight pack, `step(tok, pos)` returns the fp32
logits of one position, `clear_kv()` resets the cache, `launches` counts kernels.
The reference panics on CUDA errors; here every failure raises Gpt2qError with
the library's message. Batched prefill/decode/greedy generation and device-side
multi-step decode are the additions this B200 build is for.
"""
from __future__ import annotations

import ctypes as C
import json

import numpy as np

from . import _ffi
from .pack import Meta, Pack


def _descs(pack: Pack):
    arr = (_ffi.TensorDesc * len(pack.tensors))()
    keep = []
    for i, (name, t) in enumerate(pack.tensors.items()):
        data = np.ascontiguousarray(t.data)
        keep.append(data)
        nb, ab = name.encode(), t.atom.encode()
        keep += [nb, ab]
        arr[i].name = nb
        arr[i].atom = ab
        arr[i].ndim = len(t.shape)
        for k, s in enumerate(t.shape):
            arr[i].shape[k] = s
        arr[i].data = data.ctypes.data
        arr[i].len = data.nbytes
    return arr, keep


def _page_table(table) -> _ffi.PageTable:
    """A tensor [rows, pages] as the C structure. One row may have any stride; rows that share storage (an expanded
    table, overlapping windows) keep theirs, which is below the width and refused by the call."""
    rows, width = table.shape
    return _ffi.PageTable(table.data_ptr(), rows, width, table.stride(0) if rows > 1 else max(table.stride(0), width))


class Gpu:
    def __init__(self, pack: Pack, device: int = 0, max_seqs: int = 1, max_tokens: int = 0,
                 tp_size: int = 1, tp_rank: int = 0, nccl_id: bytes | None = None):
        self._lib = _ffi.load()
        self.meta = pack.meta
        cfg = _ffi.Config(pack.meta.n_embd, pack.meta.n_layer, pack.meta.n_head, pack.meta.n_ctx,
                          pack.meta.vocab, pack.meta.ln_eps, max_seqs, max_tokens)
        descs, keep = _descs(pack)
        h = C.c_void_p()
        if tp_size > 1:
            if nccl_id is None or len(nccl_id) != 128:
                raise ValueError("tensor-parallel Gpu needs the 128-byte NCCL unique id")
            idbuf = C.create_string_buffer(bytes(nccl_id), 128)
            rc = self._lib.gpt2q_create_tp(C.byref(cfg), descs, len(pack.tensors), device, tp_size, tp_rank,
                                           idbuf, C.byref(h))
        else:
            rc = self._lib.gpt2q_create(C.byref(cfg), descs, len(pack.tensors), device, C.byref(h))
        del keep
        _ffi.check(self._lib, None, rc)
        self.h = h
        self.max_seqs = max_seqs
        self.device = device

    @classmethod
    def from_smt(cls, path: str, device: int = 0, max_seqs: int = 1, max_tokens: int = 0,
                 verify: bool = True) -> "Gpu":
        """Engine::load + Gpu::new (gpt2.rs:43-89, gpu.rs:75-157) straight from an SMT file:
        the library maps the file, verifies the merkle content_id and every tensor digest
        (unless verify=False) and uploads the tensors; any mismatch raises Gpt2qError."""
        from .smt import inspect
        arch = inspect(path, verify=False)["arch"]
        self = cls.__new__(cls)
        self._lib = _ffi.load()
        self.meta = Meta(arch["n_embd"], arch["n_layer"], arch["n_head"], arch["n_ctx"], arch["vocab_size"])
        h = C.c_void_p()
        rc = self._lib.gpt2q_create_from_smt(str(path).encode(), device, max_seqs, max_tokens, 1 if verify else 0,
                                             C.byref(h))
        _ffi.check(self._lib, None, rc)
        self.h = h
        self.max_seqs = max_seqs
        self.device = device
        return self

    # ---- lifetime ----
    def close(self):
        if getattr(self, "h", None):
            self._lib.gpt2q_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _check(self, rc: int):
        _ffi.check(self._lib, self.h, rc)

    # ---- reference-shaped API (gpu.rs) ----
    def step(self, tok: int, pos: int) -> np.ndarray:
        """Gpu::step (gpu.rs:212): one token of sequence slot 0 -> vocab logits."""
        out = np.empty(self.meta.vocab, dtype=np.float32)
        self._check(self._lib.gpt2q_step(self.h, int(tok), int(pos), out.ctypes.data_as(_ffi._f32p)))
        return out

    def clear_kv(self, slots=None):
        """Gpu::clear_kv (gpu.rs:203)."""
        if slots is None:
            self._check(self._lib.gpt2q_reset_kv(self.h, None, 0))
        else:
            s = np.ascontiguousarray(slots, dtype=np.int32)
            self._check(self._lib.gpt2q_reset_kv(self.h, s.ctypes.data_as(_ffi._i32p), s.size))

    @property
    def launches(self) -> int:
        return int(self._lib.gpt2q_launches(self.h))

    # ---- batched API ----
    def decode(self, tok, pos, slots=None, want_logits: bool = False):
        tok = np.ascontiguousarray(tok, dtype=np.uint32)
        pos = np.ascontiguousarray(pos, dtype=np.int32)
        n = tok.size
        sl = None if slots is None else np.ascontiguousarray(slots, dtype=np.int32)
        nxt = np.empty(n, dtype=np.uint32)
        lg = np.empty((n, self.meta.vocab), dtype=np.float32) if want_logits else None
        self._check(self._lib.gpt2q_decode(
            self.h, tok.ctypes.data, pos.ctypes.data, None if sl is None else sl.ctypes.data, n,
            None if lg is None else lg.ctypes.data, nxt.ctypes.data))
        return (nxt, lg) if want_logits else nxt

    @staticmethod
    def _flatten(prompts):
        prompts = [np.ascontiguousarray(p, dtype=np.uint32) for p in prompts]
        offs = np.zeros(len(prompts) + 1, dtype=np.int32)
        offs[1:] = np.cumsum([p.size for p in prompts])
        toks = np.concatenate(prompts) if prompts else np.zeros(0, np.uint32)
        return np.ascontiguousarray(toks, dtype=np.uint32), offs

    def prefill(self, prompts, slots=None, want_logits: bool = False):
        toks, offs = self._flatten(prompts)
        n = len(prompts)
        sl = None if slots is None else np.ascontiguousarray(slots, dtype=np.int32)
        nxt = np.empty(n, dtype=np.uint32)
        lg = np.empty((n, self.meta.vocab), dtype=np.float32) if want_logits else None
        self._check(self._lib.gpt2q_prefill(
            self.h, toks.ctypes.data_as(_ffi._u32p), offs.ctypes.data_as(_ffi._i32p),
            None if sl is None else sl.ctypes.data_as(_ffi._i32p), n,
            None if lg is None else lg.ctypes.data_as(_ffi._f32p), nxt.ctypes.data_as(_ffi._u32p)))
        return (nxt, lg) if want_logits else nxt

    def decode_steps(self, steps: int, n_seq: int, want_tokens: bool = True):
        out = np.empty((steps, n_seq), dtype=np.uint32) if want_tokens else None
        self._check(self._lib.gpt2q_decode_steps(
            self.h, int(steps), None if out is None else out.ctypes.data_as(_ffi._u32p)))
        return out

    def generate_greedy(self, prompts, steps: int) -> np.ndarray:
        """generate_greedy (gpt2.rs:367-388) for every prompt; returns [n_seq, steps]."""
        toks, offs = self._flatten(prompts)
        out = np.empty((len(prompts), steps), dtype=np.uint32)
        self._check(self._lib.gpt2q_generate_greedy(
            self.h, toks.ctypes.data_as(_ffi._u32p), offs.ctypes.data_as(_ffi._i32p), len(prompts), int(steps),
            out.ctypes.data_as(_ffi._u32p)))
        return out

    def set_adapter(self, a, b):
        """Publish a post-ln_f adapter h += B (A h) (Gpu::set_adapter, gpu.rs:188-194):
        a [r, d], b [d, r] float32; later steps use it."""
        a = np.ascontiguousarray(a, dtype=np.float32)
        b = np.ascontiguousarray(b, dtype=np.float32)
        r = a.shape[0]
        if a.shape != (r, self.meta.n_embd) or b.shape != (self.meta.n_embd, r):
            raise ValueError("adapter shapes must be a [r, d] and b [d, r]")
        self._check(self._lib.gpt2q_set_adapter(self.h, a.ctypes.data_as(_ffi._f32p), b.ctypes.data_as(_ffi._f32p),
                                                int(r)))

    def clear_adapter(self):
        self._check(self._lib.gpt2q_clear_adapter(self.h))

    def nll(self, ids, slot: int = 0) -> float:
        """Teacher-forced NLL per token (nll_per_token, gpt2.rs:347-364), computed on the
        device; overwrites the KV cache of `slot`."""
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        out = C.c_double(0.0)
        self._check(self._lib.gpt2q_nll(self.h, ids.ctypes.data_as(_ffi._u32p), int(ids.size), int(slot),
                                        C.byref(out)))
        return float(out.value)

    def trunk_input_grad(self, ids, dlogits):
        """(dx [n][n_embd], lnf_out [n][n_embd]): the trunk input gradient of trunk_input_grad
        (gpu_backward.rs:651-790) for dlogits [n][vocab], forward and backward on the device."""
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        n = ids.size
        dl = np.ascontiguousarray(dlogits, dtype=np.float32)
        if dl.shape != (n, self.meta.vocab):
            raise ValueError(f"dlogits must be [{n}][{self.meta.vocab}]")
        dx = np.empty((n, self.meta.n_embd), np.float32)
        lnf = np.empty((n, self.meta.n_embd), np.float32)
        self._check(self._lib.gpt2q_trunk_input_grad(self.h, ids.ctypes.data_as(_ffi._u32p), n,
                                                     dl.ctypes.data_as(_ffi._f32p), dx.ctypes.data_as(_ffi._f32p),
                                                     lnf.ctypes.data_as(_ffi._f32p)))
        return dx, lnf

    def score(self, ids, top: int = 0, slot: int = 0):
        """Log probabilities of ids[1:] under the model, the entropies, and the `top` likeliest tokens at
        every position: (lp [n-1], entropy [n-1], top_ids [n-1][top], top_lp [n-1][top]); overwrites the
        KV cache of `slot`, as nll does."""
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        rows = max(0, ids.size - 1)
        lp, ent = np.empty(rows, np.float32), np.empty(rows, np.float32)
        top_ids, top_lp = np.empty((rows, max(0, top)), np.int32), np.empty((rows, max(0, top)), np.float32)
        self._check(self._lib.gpt2q_score(self.h, ids.ctypes.data, int(ids.size), int(slot), int(top), lp.ctypes.data,
                                          ent.ctypes.data, top_ids.ctypes.data, top_lp.ctypes.data))
        return lp, ent, top_ids, top_lp

    def trunk_score_grad(self, ids, targets, d_lp=None, d_entropy=None):
        """trunk_input_grad for the loss sum(d_lp * lp + d_entropy * entropy) over the positions' log
        probabilities of `targets` (negative: none) and entropies, all on the device. Returns (dx, lnf_out, lp,
        entropy)."""
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        n, d = ids.size, self.meta.n_embd
        tgt = np.ascontiguousarray(targets, dtype=np.int32)
        grads = [None if g is None else np.ascontiguousarray(g, dtype=np.float32) for g in (d_lp, d_entropy)]
        if tgt.shape != (n,) or any(g is not None and g.shape != (n,) for g in grads):
            raise ValueError(f"targets, d_lp and d_entropy must have {n} elements")
        dx, lnf = np.empty((n, d), np.float32), np.empty((n, d), np.float32)
        lp, ent = np.empty(n, np.float32), np.empty(n, np.float32)
        g0, g1 = (None if g is None else g.ctypes.data for g in grads)
        self._check(self._lib.gpt2q_trunk_score_grad(self.h, ids.ctypes.data, n, tgt.ctypes.data, g0, g1, lp.ctypes.data,
                                                     ent.ctypes.data, dx.ctypes.data, lnf.ctypes.data))
        return dx, lnf, lp, ent

    # ---- decode over paged caches (smelt_b200.paged.PagedKV, one per layer) ----
    def _paged(self, layers, table):
        import torch

        if len(layers) != self.meta.n_layer or any(kv.index != self.device for kv in layers):
            raise ValueError(f"{self.meta.n_layer} paged caches on device {self.device} are needed, one per layer")
        if (not table.is_cuda or table.get_device() != self.device or table.dtype != torch.int32 or table.dim() != 2
                or table.stride(1) != 1):
            raise ValueError(f"table must be int32 [rows, pages] on cuda:{self.device}")
        # what torch has queued (the pools, the table) comes before this handle's stream
        torch.cuda.current_stream(self.device).synchronize()
        return (_ffi.PagedKV * len(layers))(*(kv.c for kv in layers)), _page_table(table)

    def page_out(self, slot: int, n_tokens: int, layers, table, row: int):
        """Copies the first n_tokens cached positions of arena slot `slot` into row `row` of `table` of every
        layer's paged cache."""
        arr, t = self._paged(layers, table)
        self._check(self._lib.gpt2q_page_out(self.h, int(slot), int(n_tokens), arr, C.byref(t), int(row)))

    def decode_paged(self, tok, pos, layers, table, want_logits: bool = False):
        """decode() over paged caches: sequence i is row i of `table`."""
        tok = np.ascontiguousarray(tok, dtype=np.uint32)
        pos = np.ascontiguousarray(pos, dtype=np.int32)
        n = tok.size
        if pos.size != n:
            raise ValueError("tok and pos must have the same length")
        nxt = np.empty(n, dtype=np.uint32)
        lg = np.empty((n, self.meta.vocab), dtype=np.float32) if want_logits else None
        arr, t = self._paged(layers, table)
        self._check(self._lib.gpt2q_decode_paged(self.h, tok.ctypes.data, pos.ctypes.data, n, arr, C.byref(t),
                                                 None if lg is None else lg.ctypes.data, nxt.ctypes.data))
        return (nxt, lg) if want_logits else nxt

    def dequant(self, name: str, numel: int) -> np.ndarray:
        out = np.empty(numel, dtype=np.float32)
        self._check(self._lib.gpt2q_dequant(self.h, name.encode(), out.ctypes.data_as(_ffi._f32p), numel))
        return out

    # ---- plumbing ----
    def set_stream(self, stream_handle: int | None):
        self._check(self._lib.gpt2q_set_stream(self.h, C.c_void_p(stream_handle or 0)))

    def sync(self):
        self._check(self._lib.gpt2q_sync(self.h))

    def profile(self, enable: bool):
        self._check(self._lib.gpt2q_profile(self.h, 1 if enable else 0))

    def profile_kernels(self, reps: int = 20) -> dict:
        """Steady-state per-launch time of every kernel type of one decode step."""
        buf = C.create_string_buffer(1 << 16)
        self._check(self._lib.gpt2q_profile_kernels(self.h, int(reps), buf, len(buf)))
        return json.loads(buf.value.decode())

    def info(self) -> dict:
        """Execution paths of this handle (persistent single-sequence decode, tensor cores)."""
        buf = C.create_string_buffer(1 << 20)
        self._check(self._lib.gpt2q_info(self.h, buf, len(buf)))
        return json.loads(buf.value.decode())

    def profile_read(self) -> dict:
        buf = C.create_string_buffer(1 << 16)
        self._check(self._lib.gpt2q_profile_read(self.h, buf, len(buf)))
        return json.loads(buf.value.decode())
