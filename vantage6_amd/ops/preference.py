"""Losses on the log-probabilities of given tokens (csrc/lm_loss.hip).

Federated alignment: stations that hold preferences or rewarded answers
train on them locally. Both losses read the model's logits once for the row
statistics (maximum and sum) and once for the gradient, which needs no
[rows, V] temporary beside the result:

- ``preference_loss``: with s the log-probability of a whole answer,
  r = beta (s - s_ref), z = r_chosen - r_rejected, the loss of a pair is
  -(1 - e) log sigmoid(z) - e log sigmoid(-z);
- ``policy_loss``: with the ratio rho = exp(lp - lp_old) of a token, its loss
  is -min(rho A, clip(rho, 1 - low, 1 + high) A) + kl_coef * KL, where KL =
  exp(lp_ref - lp) - (lp_ref - lp) - 1.

The frozen model's log-probabilities are constants; per token they are
``-cross_entropy(logits, targets, reduction="none")``.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import hip_ops
from .lm_logits import (check_logits, check_mask, check_reduction, check_rows,
                        fold, kernel_rows, reduce_rows, reference_dtype)


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor  # scalar, or [N]
    chosen_rewards: torch.Tensor  # [N] float32, detached
    rejected_rewards: torch.Tensor  # [N] float32, detached


class PolicyLoss(NamedTuple):
    loss: torch.Tensor  # scalar, or [...]
    logps: torch.Tensor  # [...] float32, detached; 0 where masked
    kl: torch.Tensor  # [...] float32, detached; 0 where masked


def _token_logps(logits, targets, live):
    """CPU path: log-probability of each target, 0 where not ``live``; a
    target outside the row gives NaN."""
    V = logits.shape[-1]
    x = torch.where(live[..., None], logits, 0).to(reference_dtype(logits))
    lp = torch.log_softmax(x, -1).gather(-1, targets.clamp(0, V - 1)[..., None])[..., 0]
    lp = lp * torch.where((targets < 0) | (targets >= V), float("nan"), 1.0)
    return torch.where(live, lp, 0.0).double()


def preference_loss(logits: torch.Tensor, targets: torch.Tensor,
                    ref_logps: torch.Tensor, *, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100,
                    reduction: str = "mean") -> PreferenceLoss:
    """Paired log-ratio loss of N chosen against N rejected answers.

    ``logits`` is ``[2N, T, V]``, the chosen answers first, row n paired with
    row N + n; ``targets`` ``[2N, T]`` the token that each row of logits
    predicts (already shifted), ``ignore_index`` where none counts (prompt and
    padding: their logits are not read and get an exactly zero gradient);
    ``ref_logps`` ``[2N]`` the frozen model's sums over each answer, fp32 or
    fp64. A target outside [0, V) makes its pair NaN.

    ``reduction``: "mean" over the pairs, "sum", or "none" (``[N]``)."""
    check_logits(logits)
    red = check_reduction(reduction)
    if logits.dim() != 3 or logits.shape[0] % 2:
        raise ValueError("logits must be [2N, T, V], chosen answers first, got "
                         f"{tuple(logits.shape)}")
    if logits.shape[0] and not logits.shape[1]:
        raise ValueError("answers must have at least one position")
    check_rows("targets", targets, logits, logits.shape[:2], False)
    check_rows("ref_logps", ref_logps, logits, logits.shape[:1], True)
    if not (math.isfinite(beta) and beta > 0):
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0 <= label_smoothing < 0.5:
        raise ValueError(f"label_smoothing must be in [0, 0.5), got {label_smoothing}")
    n = logits.shape[0] // 2
    if logits.is_cuda:
        return PreferenceLoss(*hip_ops().lm_preference_loss(
            kernel_rows(logits), targets, ref_logps, beta, label_smoothing,
            ignore_index, red))
    targets = targets.long()
    lp = _token_logps(logits, targets, targets != ignore_index)
    r = beta * (lp.sum(-1) - ref_logps.double())
    z = r[:n] - r[n:]
    rows = -(1 - label_smoothing) * torch.nn.functional.logsigmoid(z)
    if label_smoothing:
        rows = rows - label_smoothing * torch.nn.functional.logsigmoid(-z)
    loss = reduce_rows(rows, None, reduction)
    if logits.dtype != torch.float64:
        loss = loss.float()
    r = r.detach().float()
    return PreferenceLoss(loss, r[:n], r[n:])


def policy_loss(logits: torch.Tensor, actions: torch.Tensor,
                old_logps: torch.Tensor, advantages: torch.Tensor,
                ref_logps: torch.Tensor | None = None, *,
                mask: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0,
                reduction: str = "mean") -> PolicyLoss:
    """Clipped policy loss of sampled tokens, with a KL term.

    ``logits`` is ``[..., V]``; ``actions`` the sampled tokens, ``old_logps``
    their log-probabilities when they were sampled, ``advantages``, and
    ``ref_logps`` the frozen model's (None: no KL term; with ``kl_coef`` 0 the
    KL is reported only), all ``[...]``.
    Tokens where ``mask`` is False do not count: their logits are not read,
    loss, ``logps``, ``kl`` and gradient are exactly 0. The gradient passes
    where the ratio sits on a border of the clip. An action outside [0, V)
    makes its token NaN.

    ``reduction``: "mean" over the tokens that count, "sum", or "none"."""
    check_logits(logits)
    red = check_reduction(reduction)
    shape = logits.shape[:-1]
    check_rows("actions", actions, logits, shape, False)
    check_rows("old_logps", old_logps, logits, shape, True)
    check_rows("advantages", advantages, logits, shape, True)
    if ref_logps is not None:
        check_rows("ref_logps", ref_logps, logits, shape, True)
    if mask is not None:
        check_mask(mask, logits, shape)
    if not 0 <= clip_low < 1 or not (math.isfinite(clip_high) and clip_high >= 0):
        raise ValueError("clip_low must be in [0, 1) and clip_high >= 0, got "
                         f"{clip_low}, {clip_high}")
    if not (math.isfinite(kl_coef) and kl_coef >= 0):
        raise ValueError(f"kl_coef must be >= 0, got {kl_coef}")
    if kl_coef > 0 and ref_logps is None:
        raise ValueError("kl_coef needs ref_logps")
    if logits.is_cuda:
        x = kernel_rows(logits)
        loss, logps, kl = hip_ops().lm_policy_loss(
            x, fold(actions, x), fold(old_logps, x), fold(advantages, x),
            fold(ref_logps, x), fold(mask, x), clip_low, clip_high, kl_coef, red)
        if x.dim() != logits.dim():
            logps, kl = logps.reshape(shape), kl.reshape(shape)
            loss = loss.reshape(shape) if reduction == "none" else loss
        return PolicyLoss(loss, logps, kl)
    live = torch.ones_like(actions, dtype=torch.bool) if mask is None else mask
    lp = _token_logps(logits, actions.long(), live)
    A = torch.where(live, advantages, 0).double()
    moved = lp - torch.where(live, old_logps, 0).double()
    ratio = moved.detach().exp()
    held = ratio.clamp(1 - clip_low, 1 + clip_high)
    moves = torch.where(A > 0, ~(ratio > 1 + clip_high), ~(ratio < 1 - clip_low))
    moves = moves | A.isnan()  # a NaN stays one
    # what the clip holds has no gradient, be the ratio +inf
    ratio = torch.where(moves, moved, 0.0).exp()
    rows = -torch.where(moves, ratio * A, held * A)
    kl = torch.zeros_like(lp)
    if ref_logps is not None:
        d = torch.where(live, ref_logps, 0).double() - lp
        kl = torch.expm1(d) - d
        if kl_coef:  # else it is reported only: it may be +inf
            rows = rows + kl_coef * kl
    rows = torch.where(live, rows, 0.0)
    loss = reduce_rows(rows, live, reduction)
    if logits.dtype != torch.float64:
        loss = loss.float()
    return PolicyLoss(loss, lp.detach().float(),
                      torch.where(live, kl, 0.0).detach().float())
