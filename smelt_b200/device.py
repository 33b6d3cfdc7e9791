"""Shared pieces of the operators on device memory (`paged`, `logprobs`): torch CUDA tensors in and
out, the current torch stream of the tensors' device, no synchronisation. Nothing here is recorded
by autograd; the gradients are calls of their own."""
from __future__ import annotations

import ctypes as C

import torch

from . import _ffi

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

# the raw handle of the current stream, without building a torch.cuda.Stream object per call
stream_of = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def need(ok: bool, msg: str):
    if not ok:
        raise ValueError(msg)


def on_device(t, index: int, name: str):
    """t is a tensor on CUDA device `index`."""
    if not (t.is_cuda and t.get_device() == index):
        raise ValueError(f"{name} must be a tensor on cuda:{index}")


def ints(t, index: int, name: str, n: int):
    """t is a contiguous int32 vector of n elements on CUDA device `index`."""
    on_device(t, index, name)
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements")


def call(fn, index: int, *args):
    """fn(*args, stream) with CUDA device `index` current."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream_of(index))
    if rc:
        _ffi.check(_ffi.load(), None, rc)


__all__ = ["C", "DTYPES", "call", "ints", "need", "on_device", "stream_of"]
