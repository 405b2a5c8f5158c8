"""Scores of given tokens under a model's logits: the log-softmax, the loss and
the perplexity sums of the reference (model/model.py:144-152,
evaluation/perplexity.py), with the entropy and the likeliest alternatives that
sampling and evaluation ask for, in one pass over the logits."""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import ops


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # fp32 [rows], 0 at ignored targets; differentiable
    entropy: torch.Tensor       # fp32 [rows]; differentiable
    top_logprobs: torch.Tensor  # fp32 [rows, top_k], best first
    top_ids: torch.Tensor       # int64 [rows, top_k]


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, ignore_index):
        *found, stats = ops.token_logprobs(logits, targets, top_k, ignore_index, return_stats=True)
        ctx.save_for_backward(logits, targets, stats)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(found[2], found[3])
        ctx.set_materialize_grads(False)
        return tuple(found)

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy, _top, _ids):
        logits, targets, stats = ctx.saved_tensors
        if g_logprobs is None and g_entropy is None:
            return None, None, None, None
        return ops.token_logprobs_backward(logits, targets, stats, g_logprobs, g_entropy,
                                           ctx.ignore_index), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Scores of the tokens targets [rows] (int64) under softmax(logits
    [rows,V]); logprobs and entropy are differentiable in the logits.  Rows
    whose target is ``ignore_index`` score 0 and pass no gradient to logprobs.
    top_k <= 64 alternatives, ties by lowest index."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k, ignore_index))
    return TokenLogprobs(*ops.token_logprobs(logits, targets, top_k, ignore_index))
