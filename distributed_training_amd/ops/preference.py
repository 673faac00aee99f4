"""Losses that train a language model on rewards or preferences, from its logits: token log-probabilities, the
clipped policy loss with a KL term, and the paired preference loss; each with its gradient.

They stand beside ``ops/lm.py``'s cross-entropy and take what a model's forward without targets returns: logits
``[B, S, V]`` (or ``[N, V]``) and the token ids ``[B, S]`` that each position is scored on, with ``ignore_index`` where
a position does not count (prompts, padding).  Positions that do not count -- a target of ``ignore_index`` or outside
``[0, V)`` -- have log-probability 0 and a zero gradient, whatever their logits hold.

GPU tensors take the HIP kernels of ``csrc/preference.hip`` (bf16, fp16 or fp32 logits; rows of any stride and
alignment, any vocabulary) through the autograd functions of ``csrc/bindings_pref.cpp``, which check their tensors.
CPU tensors take the same math in PyTorch, fp64 logits among them (with fp32 or fp64 per-token inputs).  Beside other
logits per-token inputs are fp32; statistics over the vocabulary are fp32, per-token terms and sums fp64.  On the GPU
each loss can be differentiated once: a gradient taken with ``create_graph`` is refused where it is differentiated.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence

import torch
import torch.nn.functional as F

from . import native


class PolicyLoss(NamedTuple):
    """``loss`` carries the gradient; the rest is detached: the tokens' log-probabilities under the current policy, the
    mean KL estimate over counted tokens (0 without a reference) and the fraction of them that the clip stopped."""

    loss: torch.Tensor
    logp: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


class PreferenceLoss(NamedTuple):
    """``loss`` carries the gradient; detached: the sequences' log-probabilities ``[2 P]`` and the pairs' margins
    ``[P]`` (positive where the chosen sequence gained more than the rejected one)."""

    loss: torch.Tensor
    logp: torch.Tensor
    margin: torch.Tensor


# ------------------------------------------------------------------ checks
def _check(logits: torch.Tensor, target: torch.Tensor) -> None:
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits must be [N, V] or [B, S, V] (got {tuple(logits.shape)})")
    if target.shape != logits.shape[:-1]:
        raise ValueError(f"target must be {tuple(logits.shape[:-1])} (got {tuple(target.shape)})")
    if logits.shape[-1] < 1:
        raise ValueError("logits must have a vocabulary")
    if target.dtype != torch.int64:
        raise TypeError(f"target must be int64 (got {target.dtype})")
    if target.device != logits.device:
        raise ValueError(f"target is on {target.device}, logits on {logits.device}")
    if not logits.dtype.is_floating_point:
        raise TypeError(f"logits must be floating point (got {logits.dtype})")


def _check_tokens(t: Optional[torch.Tensor], logits: torch.Tensor, name: str, shapes: Sequence[torch.Size]) -> None:
    if t is None:
        return
    if t.shape not in shapes:
        raise ValueError(f"{name} must be {' or '.join(str(tuple(s)) for s in shapes)} (got {tuple(t.shape)})")
    # (fp64 logits, which only the CPU takes, have fp64 log-probabilities)
    if t.dtype != torch.float32 and not (t.dtype == logits.dtype == torch.float64):
        raise TypeError(f"{name} must be float32 (got {t.dtype}, logits {logits.dtype})")
    if t.device != logits.device:
        raise ValueError(f"{name} is on {t.device}, logits on {logits.device}")


def _positive(x: float, name: str) -> float:
    if not (x > 0.0 and math.isfinite(x)):
        raise ValueError(f"{name} must be positive and finite (got {x})")
    return float(x)


def _temperature(x: float) -> float:
    if not 1e-6 <= x <= 1e6:
        raise ValueError(f"temperature must be between 1e-6 and 1e6 (got {x})")
    return float(x)


def _not_negative(x: float, name: str) -> float:
    if not (x >= 0.0 and math.isfinite(x)):
        raise ValueError(f"{name} must be finite and not negative (got {x})")
    return float(x)


# ------------------------------------------------------------------ token log-probabilities
def _live(logits: torch.Tensor, target: torch.Tensor, ignore_index: int) -> torch.Tensor:
    return (target != ignore_index) & (target >= 0) & (target < logits.shape[-1])


def token_logprobs_reference(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                             temperature: float = 1.0) -> torch.Tensor:
    """:func:`token_logprobs` in plain PyTorch, in fp32 (fp64 for fp64 logits)."""
    live = _live(logits, target, ignore_index)
    x = logits if logits.dtype == torch.float64 else logits.float()
    x = x.masked_fill(~live.unsqueeze(-1), 0.0) / temperature
    lp = torch.log_softmax(x, -1).gather(-1, torch.where(live, target, 0).unsqueeze(-1)).squeeze(-1)
    return lp.masked_fill(~live, 0.0)


def token_logprobs(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                   temperature: float = 1.0) -> torch.Tensor:
    """``log softmax(logits / temperature)`` at each position's target: fp32, of ``target``'s shape, 0 where a position
    does not count.  What a rollout stores as ``old_logp`` and a frozen model gives as ``ref_logp``; differentiable."""
    temperature = _temperature(temperature)
    if logits.is_cuda:
        return native().token_logprobs(logits, target, ignore_index, temperature)
    _check(logits, target)
    return token_logprobs_reference(logits, target, ignore_index, temperature)


# ------------------------------------------------------------------ clipped policy loss
def policy_loss_reference(logits: torch.Tensor, target: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                          ref_logp: Optional[torch.Tensor] = None, clip: float = 0.2, clip_high: Optional[float] = None,
                          kl_coef: float = 0.0, reduction: str = "token", ignore_index: int = -100,
                          temperature: float = 1.0, scale: float = 1.0) -> PolicyLoss:
    """:func:`policy_loss` in plain PyTorch."""
    live = _live(logits, target, ignore_index)
    logp = token_logprobs_reference(logits, target, ignore_index, temperature)
    lp = logp.double()
    A = advantages.double()
    A = A.unsqueeze(-1) if A.dim() < target.dim() else A
    # (inputs of positions that do not count may hold anything)
    A = A.expand(target.shape).masked_fill(~live, 0.0)
    ratio = torch.exp(lp - torch.where(live, old_logp.double(), lp.detach()))
    high = 1.0 + (clip if clip_high is None else clip_high)
    each = -torch.minimum(ratio * A, ratio.clamp(1.0 - clip, high) * A)
    clipped = ((A > 0) & (ratio > high)) | ((A < 0) & (ratio < 1.0 - clip))
    tokens = live.sum().clamp(min=1)
    kl = torch.zeros_like(lp)
    if ref_logp is not None:
        d = torch.where(live, ref_logp.double(), lp.detach()) - lp
        kl = torch.expm1(d) - d
        if kl_coef:
            each = each + kl_coef * kl
    if reduction == "token":
        loss = each.sum() / tokens
    else:
        loss = (each.sum(-1) / live.sum(-1).clamp(min=1)).sum() / max(1, target.shape[0])
    out = logp.detach() if logp.dtype == torch.float64 else logp.detach().float()
    return PolicyLoss((loss * scale).to(logp.dtype), out, (kl.detach().sum() / tokens).to(logp.dtype),
                      (clipped.sum() / tokens).to(logp.dtype))


def policy_loss(logits: torch.Tensor, target: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                ref_logp: Optional[torch.Tensor] = None, clip: float = 0.2, clip_high: Optional[float] = None,
                kl_coef: float = 0.0, reduction: str = "token", ignore_index: int = -100, temperature: float = 1.0,
                scale: float = 1.0) -> PolicyLoss:
    """The clipped policy loss of sampled tokens with a KL term::

        r = exp(lp - old_logp)
        loss = scale * mean(-min(r A, clamp(r, 1 - clip, 1 + clip_high) A) + kl_coef * (exp(d) - d - 1)),  d = ref_logp - lp

    ``lp``: :func:`token_logprobs` of the targets.  ``old_logp`` / ``ref_logp``: fp32, of ``target``'s shape, no
    gradient.  ``advantages``: the same shape, or ``[B]`` for one a sequence.  ``clip_high``: the upper bound where it
    differs from ``clip``.  ``reduction``: ``"token"`` -- the mean over all tokens that count; ``"sequence"`` -- the mean over the
    B sequences of each one's token mean (an empty sequence adds 0).  ``scale`` multiplies the loss: with gradient
    accumulation pass 1 / steps here rather than dividing the result.  No token counting: the loss is 0.

    On the GPU, from 128 tokens on and up to vocabularies of 131072 (fp32: 65536), the gradient of the logits is formed in the
    forward, in the same pass over them, and held until the backward: as much memory as the logits take."""
    clip, kl_coef = _not_negative(clip, "clip"), _not_negative(kl_coef, "kl_coef")
    clip_high = clip if clip_high is None else _not_negative(clip_high, "clip_high")
    temperature = _temperature(temperature)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite (got {scale})")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction must be 'token' or 'sequence' (got {reduction!r})")
    if reduction == "sequence" and logits.dim() == 2:
        raise ValueError("reduction='sequence' needs logits [B, S, V]")
    if kl_coef and ref_logp is None:
        raise ValueError("kl_coef needs ref_logp")
    if logits.is_cuda:
        return PolicyLoss(*native().policy_loss(logits, target, old_logp, advantages, ref_logp, clip, clip_high, kl_coef,
                                                reduction == "sequence", ignore_index, temperature, scale))
    _check(logits, target)
    for t, name in ((old_logp, "old_logp"), (ref_logp, "ref_logp")):
        _check_tokens(t, logits, name, [target.shape])
    _check_tokens(advantages, logits, "advantages", [target.shape, target.shape[:1]][:target.dim()])
    return policy_loss_reference(logits, target, old_logp.detach(), advantages.detach(),
                                 None if ref_logp is None else ref_logp.detach(), clip, clip_high, kl_coef, reduction,
                                 ignore_index, temperature, scale)


# ------------------------------------------------------------------ paired preference loss
def preference_loss_reference(logits: torch.Tensor, target: torch.Tensor, ref_logp: Optional[torch.Tensor] = None,
                              beta: float = 0.1, label_smoothing: float = 0.0, average: bool = False,
                              ignore_index: int = -100, scale: float = 1.0) -> PreferenceLoss:
    """:func:`preference_loss` in plain PyTorch."""
    live = _live(logits, target, ignore_index)
    lp = token_logprobs_reference(logits, target, ignore_index)
    total = lp.double().sum(-1)
    if average:
        total = total / live.sum(-1).clamp(min=1)
    gap = total if ref_logp is None else total - ref_logp.double()
    P = logits.shape[0] // 2
    h = beta * (gap[:P] - gap[P:])
    loss = -((1.0 - label_smoothing) * F.logsigmoid(h) + label_smoothing * F.logsigmoid(-h)).mean() * scale
    return PreferenceLoss(loss.to(lp.dtype), total.detach().to(lp.dtype), h.detach().to(lp.dtype))


def preference_loss(logits: torch.Tensor, target: torch.Tensor, ref_logp: Optional[torch.Tensor] = None,
                    beta: float = 0.1, label_smoothing: float = 0.0, average: bool = False, ignore_index: int = -100,
                    scale: float = 1.0) -> PreferenceLoss:
    """The loss of preference pairs from their log-ratios::

        L_i = sum_t lp_it  (average: divided by the tokens that count)
        h_p = beta * ((L_p - R_p) - (L_{p+P} - R_{p+P}))
        loss = scale * mean_p(-(1 - label_smoothing) log sigmoid(h_p) - label_smoothing log sigmoid(-h_p))

    ``logits`` ``[2 P, S, V]``: the P chosen sequences, then the P rejected ones in the same order (one forward over both).
    ``ref_logp`` ``[2 P]`` fp32: the frozen model's ``L`` of the same sequences, formed the same way (absent: 0).
    ``scale`` as in :func:`policy_loss`.  A sequence without tokens that count has ``L = 0``."""
    beta = _positive(beta, "beta")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1] (got {label_smoothing})")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite (got {scale})")
    if logits.is_cuda:
        return PreferenceLoss(*native().preference_loss(logits, target, ref_logp, beta, label_smoothing, average,
                                                        ignore_index, scale))
    _check(logits, target)
    if logits.dim() != 3 or logits.shape[0] < 2 or logits.shape[0] % 2:
        raise ValueError("logits must be [2 P, S, V]: P chosen sequences, then as many rejected ones "
                         f"(got {tuple(logits.shape)})")
    _check_tokens(ref_logp, logits, "ref_logp", [logits.shape[:1]])
    ref_logp = None if ref_logp is None else ref_logp.detach()
    return preference_loss_reference(logits, target, ref_logp, beta, label_smoothing, average, ignore_index, scale)
