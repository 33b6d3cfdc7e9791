"""Log probabilities of given tokens with entropy and top alternatives, and their gradient.

    r = token_logprobs(logits, targets, top=5)       # r.lp, r.entropy, r.top_ids, r.top_lp, r.stats
    dlogits = token_logprobs_grad(logits, targets, r.stats, d_lp, d_entropy)

torch CUDA tensors on the current torch stream; include/gpt2q.h (gpt2q_logprobs) states what masked
logits, empty rows, ties and negative targets give.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ffi
from .device import DTYPES, call, need, on_device

TOP_MAX = 64


class LogProbs(NamedTuple):
    lp: torch.Tensor | None        # [rows] float32; None without targets
    entropy: torch.Tensor          # [rows] float32
    top_ids: torch.Tensor | None   # [rows, top] int32; None when top is 0
    top_lp: torch.Tensor | None    # [rows, top] float32
    stats: torch.Tensor            # [rows, 3] float32, for token_logprobs_grad


def _logits(logits):
    if not logits.is_cuda or logits.dim() != 2 or logits.dtype not in DTYPES:
        raise ValueError("logits must be a CUDA tensor [rows, vocab] of float32, float16 or bfloat16")
    rows, vocab = logits.shape
    need(vocab >= 1 and (logits.stride(1) == 1 or vocab == 1), "logits must have unit stride over the vocabulary")
    ld = logits.stride(0) if rows > 1 else vocab
    need(ld >= vocab, "the rows of logits must not overlap")
    return logits.get_device(), rows, vocab, ld


def _targets(targets, index, rows):
    on_device(targets, index, "targets")
    if targets.dtype not in (torch.int32, torch.int64) or targets.shape != (rows,) or not targets.is_contiguous():
        raise ValueError(f"targets must be a contiguous int32 or int64 tensor of {rows} elements")
    return targets.data_ptr(), 1 if targets.dtype == torch.int64 else 0


def token_logprobs(logits, targets=None, top: int = 0, temperature: float = 1.0) -> LogProbs:
    """Under softmax(logits / temperature), per row: the log probability of its target, the entropy, and
    the `top` likeliest tokens (at most TOP_MAX) with their log probabilities. A negative target gives 0."""
    index, rows, vocab, ld = _logits(logits)
    dev = logits.device
    tp, wide = (None, 0) if targets is None else _targets(targets, index, rows)
    lp = None if targets is None else torch.empty(rows, dtype=torch.float32, device=dev)
    rest = torch.empty(4 * rows, dtype=torch.float32, device=dev)  # the entropy, then the statistics
    ids = tlp = None
    if top:
        ids = torch.empty((rows, top), dtype=torch.int32, device=dev)
        tlp = torch.empty((rows, top), dtype=torch.float32, device=dev)
    at = rest.data_ptr()
    call(_ffi.load().gpt2q_logprobs, index, logits.data_ptr(), DTYPES[logits.dtype], ld, rows, vocab, temperature, tp, wide,
         top, None if lp is None else lp.data_ptr(), at, at + 4 * rows, None if ids is None else ids.data_ptr(),
         None if tlp is None else tlp.data_ptr())
    return LogProbs(lp, rest[:rows], ids, tlp, rest[rows:].view(rows, 3))


def token_logprobs_grad(logits, targets, stats, d_lp, d_entropy=None, temperature: float = 1.0, out=None):
    """The gradient with respect to the logits, of their type, for the gradients d_lp and d_entropy ([rows]
    float32, either may be None) of token_logprobs' lp and entropy; `out` may be `logits` itself."""
    index, rows, vocab, ld = _logits(logits)
    tp, wide = (None, 0) if targets is None else _targets(targets, index, rows)
    need(targets is not None or d_lp is None, "d_lp without targets")
    on_device(stats, index, "stats")
    if stats.dtype != torch.float32 or stats.shape != (rows, 3) or not stats.is_contiguous():
        raise ValueError(f"stats must be a contiguous float32 tensor [{rows}, 3]")
    for name, g in (("d_lp", d_lp), ("d_entropy", d_entropy)):
        if g is not None:
            on_device(g, index, name)
            if g.dtype != torch.float32 or g.shape != (rows,) or not g.is_contiguous():
                raise ValueError(f"{name} must be a contiguous float32 tensor of {rows} elements")
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        lo = vocab
    else:
        oi, orows, ovocab, lo = _logits(out)
        need((oi, orows, ovocab) == (index, rows, vocab) and out.dtype == logits.dtype,
             "out must have the shape, type and device of logits")
    call(_ffi.load().gpt2q_logprobs_grad, index, logits.data_ptr(), DTYPES[logits.dtype], ld, rows, vocab, temperature, tp,
         wide, stats.data_ptr(), None if d_lp is None else d_lp.data_ptr(),
         None if d_entropy is None else d_entropy.data_ptr(), out.data_ptr(), lo)
    return out
