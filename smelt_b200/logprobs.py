"""Log probabilities of given tokens with entropy and top alternatives, and their gradient.

    r = token_logprobs(logits, targets, top=5)       # r.lp, r.entropy, r.top_ids, r.top_lp, r.stats
    dlogits = token_logprobs_grad(logits, targets, r.stats, d_lp, d_entropy)

torch CUDA tensors on the current torch stream. Nothing is recorded by autograd, for logits that require a
gradient either: training code calls token_logprobs_grad. include/gpt2q.h (gpt2q_logprobs) states what masked
logits, empty rows, ties and negative targets give.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .device import ops

TOP_MAX = 64


class LogProbs(NamedTuple):
    lp: torch.Tensor | None        # [rows] float32; None without targets
    entropy: torch.Tensor          # [rows] float32
    top_ids: torch.Tensor | None   # [rows, top] int32; None when top is 0
    top_lp: torch.Tensor | None    # [rows, top] float32
    stats: torch.Tensor            # [rows, 3] float32, for token_logprobs_grad


def token_logprobs(logits, targets=None, top: int = 0, temperature: float = 1.0) -> LogProbs:
    """Under softmax(logits / temperature), per row: the log probability of its target, the entropy, and
    the `top` likeliest tokens (at most TOP_MAX) with their log probabilities. A negative target gives 0."""
    return LogProbs._make(ops().logprobs(logits, targets, top, temperature))


def token_logprobs_grad(logits, targets, stats, d_lp, d_entropy=None, temperature: float = 1.0, out=None):
    """The gradient with respect to the logits, of their type, for the gradients d_lp and d_entropy ([rows]
    float32, either may be None) of token_logprobs' lp and entropy; `out` may be `logits` itself."""
    return ops().logprobs_grad(logits, targets, stats, d_lp, d_entropy, temperature, out)
