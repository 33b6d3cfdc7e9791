"""Loads the torch binding of the operators on device memory (csrc/torch_ops.cpp). Its calls take
torch CUDA tensors, go to the current torch stream of the tensors' device and do not synchronise;
nothing is recorded by autograd: the gradients are calls of their own."""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

import torch

from . import _ffi

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_PATH = os.path.join(_ffi.HERE, "_lib", "gpt2q_torch.so")
_ops = None


def ops():
    """The binding; raises if it has not been built."""
    global _ops
    if _ops is None:
        _ffi.load()  # the library it calls
        if not os.path.exists(_PATH):
            raise ImportError(f"gpt2q_torch.so not built at {_PATH}; run `python -m smelt_b200.build`")
        loader = importlib.machinery.ExtensionFileLoader("gpt2q_torch", _PATH)
        mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("gpt2q_torch", loader))
        loader.exec_module(mod)
        mod.set_error(_ffi.Gpt2qError)
        _ops = mod
    return _ops
