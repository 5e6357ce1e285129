"""Losses that a rewired model is tuned with, straight from its logits.

``token_logprobs``   log probability of each row's target
``preference_loss``  paired log ratios against a reference model
``policy_loss``      clipped policy gradient with a KL term

Each is differentiable with respect to the logits.  ``preference_loss_grad``
and ``policy_loss_grad`` return the loss and the logits' gradient from one
call, for ``logits.backward(result.dlogits)``; the policy loss then reads the
logits once and writes the gradient once.

Logits are [T, V], or [B, S, V] for B sequences of S rows; views whose last
axis is contiguous are read in place (``logits[:, :-1]``).  Targets are int64
of the leading shape; a row whose target is ``ignore_index`` takes no part:
its log probability and its gradient are 0.  A target outside [0, V) and a row
without a finite logit give NaN.  Log probabilities, losses and all sums are
fp32 or wider; the gradient has the logits' type.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi as C

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class PreferenceResult(NamedTuple):
    loss: torch.Tensor
    """fp32 scalar."""
    logprobs: torch.Tensor
    """fp32, the targets' shape; 0 where ignored.  Carries no gradient."""
    margins: torch.Tensor
    """fp32 [pairs]: beta times the difference of the pair's log ratios.  Carries no gradient."""
    dlogits: torch.Tensor | None = None
    """The logits' gradient (preference_loss_grad), else None."""


class PolicyResult(NamedTuple):
    loss: torch.Tensor
    """fp32 scalar."""
    logprobs: torch.Tensor
    """fp32, the targets' shape; 0 where ignored.  Carries no gradient."""
    kl: torch.Tensor
    """fp32 scalar: the KL estimate (0 without ref_logprobs).  Carries no gradient."""
    dlogits: torch.Tensor | None = None
    """The logits' gradient (policy_loss_grad), else None."""


# ----------------------------------------------------------------- checks --
def _check_rows(logits, targets):
    if logits.dtype not in _FLOATS:
        raise ValueError(f"unsupported logits dtype {logits.dtype}; expected float32, float16 or "
                         "bfloat16")
    if logits.ndim not in (2, 3):
        raise ValueError(f"logits must be [T, V] or [B, S, V], got shape {tuple(logits.shape)}")
    if logits.shape[-1] == 0:
        raise ValueError("logits need at least one class")
    if targets.dtype != torch.int64:
        raise ValueError(f"targets must be int64, got {targets.dtype}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(logits.shape[:-1])}, got "
                         f"{tuple(targets.shape)}")


def _check_per_token(name, t, targets):
    if t.shape != targets.shape:
        raise ValueError(f"{name} must have the targets' shape {tuple(targets.shape)}, got "
                         f"{tuple(t.shape)}")
    if not t.is_floating_point():
        raise ValueError(f"{name} must be floating point, got {t.dtype}")


def _inverse(denominator) -> float:
    # its inverse is an fp32 argument of the kernels, where 0 means the number of tokens
    if not 2.0 ** -126 <= denominator <= 2.0 ** 126:
        raise ValueError(f"denominator must be positive, and its inverse an fp32 number, got "
                         f"{denominator}")
    return 1.0 / float(denominator)


def _check_preference(logits, targets, ref_logprobs, cu_seqlens, label_smoothing, denominator):
    """(pairs, inverse denominator)"""
    _check_rows(logits, targets)
    _check_per_token("ref_logprobs", ref_logprobs, targets)
    if cu_seqlens is None:
        if logits.ndim != 3:
            raise ValueError("logits of shape [T, V] need cu_seqlens")
        sequences = logits.shape[0]
    else:
        if cu_seqlens.dtype not in (torch.int32, torch.int64) or cu_seqlens.ndim != 1:
            raise ValueError("cu_seqlens must be a 1-D int32 or int64 tensor")
        sequences = cu_seqlens.shape[0] - 1
    if sequences < 2 or sequences % 2:
        raise ValueError(f"sequences come in pairs (chosen, rejected): got {max(sequences, 0)}")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1), got {label_smoothing}")
    pairs = sequences // 2
    return pairs, _inverse(pairs if denominator is None else denominator)


def _check_policy(logits, targets, old_logprobs, advantages, ref_logprobs, clip_low, clip_high,
                  kl_coef, denominator):
    _check_rows(logits, targets)
    _check_per_token("old_logprobs", old_logprobs, targets)
    _check_per_token("advantages", advantages, targets)
    if ref_logprobs is not None:
        _check_per_token("ref_logprobs", ref_logprobs, targets)
    elif kl_coef != 0.0:
        raise ValueError("kl_coef needs ref_logprobs")
    if not 0.0 <= clip_low <= 1.0:
        raise ValueError(f"clip_low must be in [0, 1], got {clip_low}")
    if not clip_high >= 0.0:
        raise ValueError(f"clip_high must be >= 0, got {clip_high}")
    return 0.0 if denominator is None else _inverse(denominator)


# ------------------------------------------------------ log probabilities --
class _LogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ignore_index):
        logp, stats = C.host().token_logprobs(logits, targets, ignore_index)
        ctx.save_for_backward(logits, targets, stats)
        ctx.ignore_index = ignore_index
        return logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d):
        logits, targets, stats = ctx.saved_tensors
        grad = C.host().logits_grad(logits, targets, ctx.ignore_index, stats, d, None, None)
        return grad, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *,
                   ignore_index: int = -100) -> torch.Tensor:
    """fp32 log softmax of `logits` at `targets` (0 where ignored), the targets' shape."""
    _check_rows(logits, targets)
    return _LogprobsFn.apply(logits, targets, int(ignore_index))


# ------------------------------------------------------------- preference --
class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, ref, cu, pairs, beta, smoothing, inv_d, ignore_index):
        loss, logp, margins, _, records = C.host().preference(
            logits, targets, ignore_index, ref, cu, pairs, beta, smoothing, inv_d, 1.0, False)
        ctx.save_for_backward(logits, targets, records)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(logp, margins)
        return loss, logp, margins

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d, _logp, _margins):
        logits, targets, records = ctx.saved_tensors
        grad = C.host().logits_grad(logits, targets, ctx.ignore_index, records, None, d, None)
        return (grad,) + (None,) * 8


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor,
                    cu_seqlens: torch.Tensor | None = None, *, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100,
                    denominator: float | None = None) -> PreferenceResult:
    """Paired preference loss.

    Sequence s is rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 of [T, V] logits
    (or row s of [B, S, V] logits when cu_seqlens is None); sequences 2b and
    2b + 1 are pair b's chosen and rejected answers.  With R_s the sum over
    the sequence of logprobs - ref_logprobs and z_b = beta (R_2b - R_2b+1),

        loss = 1/D sum_b (1 - e) softplus(-z_b) + e softplus(z_b)

    e = label_smoothing, D = denominator (default: the number of pairs; give
    the whole batch's number where gradients are accumulated)."""
    pairs, inv_d = _check_preference(logits, targets, ref_logprobs, cu_seqlens, label_smoothing,
                                     denominator)
    return PreferenceResult(*_PreferenceFn.apply(
        logits, targets, ref_logprobs, cu_seqlens, pairs, float(beta), float(label_smoothing),
        inv_d, int(ignore_index)))


def preference_loss_grad(logits: torch.Tensor, targets: torch.Tensor, ref_logprobs: torch.Tensor,
                         cu_seqlens: torch.Tensor | None = None, *, beta: float = 0.1,
                         label_smoothing: float = 0.0, ignore_index: int = -100,
                         denominator: float | None = None,
                         grad_scale: float = 1.0) -> PreferenceResult:
    """``preference_loss`` and, in ``dlogits``, grad_scale times its gradient."""
    pairs, inv_d = _check_preference(logits, targets, ref_logprobs, cu_seqlens, label_smoothing,
                                     denominator)
    return PreferenceResult(*C.host().preference(
        logits, targets, int(ignore_index), ref_logprobs, cu_seqlens, pairs, beta, label_smoothing,
        inv_d, grad_scale, True)[:4])


# ----------------------------------------------------------------- policy --
class _PolicyFn(torch.autograd.Function):
    """The forward also writes the gradient for an upstream of 1, which is what
    an unscaled loss is differentiated with; the backward checks that on the
    device and computes it anew from the logits otherwise."""

    @staticmethod
    def forward(ctx, logits, targets, old, adv, ref, lo, hi, kl_coef, inv_d, ignore_index):
        loss, logp, kl, dlogits, records = C.host().policy(
            logits, targets, ignore_index, old, adv, ref, lo, hi, kl_coef, inv_d, 1.0,
            ctx.needs_input_grad[0])
        ctx.save_for_backward(logits, targets, records)
        ctx.ignore_index, ctx.dlogits = ignore_index, dlogits
        ctx.mark_non_differentiable(logp, kl)
        return loss, logp, kl

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d, _logp, _kl):
        logits, targets, records = ctx.saved_tensors
        # handed over once: a second backward over a kept graph computes its own
        ready, ctx.dlogits = ctx.dlogits, None
        grad = C.host().logits_grad(logits, targets, ctx.ignore_index, records, None, d, ready)
        return (grad,) + (None,) * 9


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                advantages: torch.Tensor, *, ref_logprobs: torch.Tensor | None = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                ignore_index: int = -100, denominator: float | None = None) -> PolicyResult:
    """Clipped policy loss with a KL term, over the tokens that count:

        r = exp(logprobs - old_logprobs)
        k = expm1(ref_logprobs - logprobs) - (ref_logprobs - logprobs)
        loss = 1/D sum kl_coef k - min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)

    D = denominator (default: the number of tokens that count; give the whole
    batch's number where gradients are accumulated).  Without such a token the
    loss and its gradient are 0.

    The gradient is written with the loss, for a loss that is differentiated as it
    is.  One that is scaled (a GradScaler's, a weight, a division) has it computed
    a second time in the backward: ``policy_loss_grad`` takes that scale and
    computes it once."""
    inv_d = _check_policy(logits, targets, old_logprobs, advantages, ref_logprobs, clip_low,
                          clip_high, kl_coef, denominator)
    return PolicyResult(*_PolicyFn.apply(
        logits, targets, old_logprobs, advantages, ref_logprobs, float(clip_low),
        float(clip_high), float(kl_coef), inv_d, int(ignore_index)))


def policy_loss_grad(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor,
                     advantages: torch.Tensor, *, ref_logprobs: torch.Tensor | None = None,
                     clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                     ignore_index: int = -100, denominator: float | None = None,
                     grad_scale: float = 1.0) -> PolicyResult:
    """``policy_loss`` and, in ``dlogits``, grad_scale times its gradient."""
    inv_d = _check_policy(logits, targets, old_logprobs, advantages, ref_logprobs, clip_low,
                          clip_high, kl_coef, denominator)
    return PolicyResult(*C.host().policy(
        logits, targets, int(ignore_index), old_logprobs, advantages, ref_logprobs, clip_low,
        clip_high, kl_coef, inv_d, grad_scale, True)[:4])
