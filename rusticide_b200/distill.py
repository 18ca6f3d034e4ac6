"""Training a draft model on the tokens its target model prefers.

`distill_loss` is the differentiable form of the engine's distillation call: the teacher's rows are
given as the survivors and log-probabilities that `Engine.sample_ex(..., logprobs=True)` lists for
them, the student's as logits. Drafts of a student trained this way are what `Engine.verify` accepts
more of. The reference (crates/rusticide-model) serves models and trains none; nothing there
corresponds to this module.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from .sampler import Engine, engine


def _engine_of(logits: torch.Tensor) -> Engine:
    if not logits.is_cuda:
        raise RuntimeError("distill_loss needs logits on a CUDA device; there is no CPU fallback")
    return engine(logits.get_device())


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, n, temperature, tail):
        loss, state = _engine_of(logits).distill_forward(logits, ids, logprobs, n, temperature, tail)
        ctx.save_for_backward(logits, ids, logprobs, n, state)
        ctx.how = (temperature, tail)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, ids, logprobs, n, state = ctx.saved_tensors
        grad = _engine_of(logits).distill_backward(
            logits, ids, logprobs, state, grad_loss.contiguous(), n, *ctx.how)
        return grad, None, None, None, None, None


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor,
                 n: Optional[torch.Tensor] = None, temperature: float = 1.0,
                 tail: bool = False) -> torch.Tensor:
    """Loss of every row of student logits [..., vocab] against a teacher's top tokens ids
    [..., top] int32 with log-probabilities logprobs [..., top] f32 (see rsc_distill in the C
    header), n [...] int32 of them a row (None: all; below 0: none). A count above `top` reads as
    `top`, as the lists of a sample_ex call have it whose survivor_cap was too small for a row: they
    hold the first ids of its survivors, not the likeliest, so give that call slots for all.
    Returns [...] f32; differentiable once, with respect to the logits. A training loop that knows each row's weight beforehand takes
    `Engine.distill_step`, which gives loss and gradient in one pass."""
    if (forward_ad.unpack_dual(logits).tangent is not None
            or forward_ad.unpack_dual(logprobs).tangent is not None):
        raise NotImplementedError("distill_loss has no forward-mode derivative")
    if logits.requires_grad and torch.is_grad_enabled():
        return _DistillLoss.apply(logits, ids, logprobs, n, temperature, tail)
    return _engine_of(logits).distill_forward(logits, ids, logprobs, n, temperature, tail,
                                                 want_state=False)[0]
