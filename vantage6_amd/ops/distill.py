"""Distillation from a teacher's top logits (csrc/lm_loss.hip).

Federated distillation: stations do not exchange weights but what their
models answer on a public set. A full row of 128256 bf16 logits is 256 KB;
``topk_logits`` makes a record of its ``k`` largest values, their places
and the row's logsumexp (under 1 KB at k = 64), and ``distill_loss`` trains
a student on such records.

With q the student's probabilities at the temperature t and p a record's,

- without ``teacher_lse``: p = softmax(values / t) over the record, and the
  loss of a row is KL(p || q);
- with it: p_k = exp(values_k / t - teacher_lse), and what the record leaves
  out, 1 - sum p, is compared as one lump with the student's mass outside the
  record's places.

Both times t**2, so that gradients keep their size over temperatures. The
upstream framework has no losses (compute lives in user images).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import hip_ops
from .lm_logits import (check_logits, check_mask,
                        check_reduction, check_rows, check_temperature, fold,
                        kernel_rows, reduce_rows, reference_dtype)

MOST_K = 256


class TopLogits(NamedTuple):
    """A row's ``k`` largest logits, largest first, and the row's logsumexp."""

    values: torch.Tensor  # [..., k], the logits' dtype
    indices: torch.Tensor  # [..., k] int64
    logsumexp: torch.Tensor  # [...] float32, of logits / temperature


@torch.no_grad()
def topk_logits(logits: torch.Tensor, k: int, temperature: float = 1.0
                ) -> TopLogits:
    """The ``k`` largest logits of each row of ``[..., V]``, with their places.

    Equal logits go to the lower index; a NaN counts as the largest. 1 <= k <=
    min(V, 256). ``logsumexp`` is that of ``logits / temperature``, as
    ``distill_loss`` takes it. The record is a constant: no gradient."""
    check_logits(logits)
    check_temperature(temperature)
    if not 1 <= k <= min(MOST_K, logits.shape[-1]):
        raise ValueError(f"k must be between 1 and min(V, {MOST_K}), got {k}")
    if logits.is_cuda:
        x = kernel_rows(logits)
        values, indices, lse = hip_ops().lm_topk(x, k, temperature)
        if logits.dim() > 3:
            rows = logits.shape[:-1]
            values, indices = values.reshape(*rows, k), indices.reshape(*rows, k)
            lse = lse.reshape(rows)
        return TopLogits(values, indices, lse)
    indices = torch.sort(logits, dim=-1, descending=True, stable=True
                         ).indices[..., :k].contiguous()
    x = logits.to(reference_dtype(logits))
    return TopLogits(logits.gather(-1, indices), indices,
                     torch.logsumexp(x / temperature, -1).float())


def distill_loss(logits: torch.Tensor, teacher_values: torch.Tensor,
                 teacher_indices: torch.Tensor,
                 teacher_lse: torch.Tensor | None = None, *,
                 temperature: float = 1.0, mask: torch.Tensor | None = None,
                 reduction: str = "mean",
                 teacher_temperature: torch.Tensor | None = None) -> torch.Tensor:
    """Divergence of ``logits`` ``[..., V]`` from a teacher's records, fp32.

    ``teacher_values`` and ``teacher_indices`` are ``[..., k]`` with k <= 256,
    in any order, ``teacher_lse`` ``[...]`` or None (see above); ``logits /
    temperature`` is what both sides are compared at. An entry with a negative
    index is absent, one with a value of -inf has no probability; the same
    index twice adds up. A row is ignored (loss 0, gradient exactly 0, whatever
    its logits hold) where ``mask`` is False, and then its logits are not read,
    or where its record holds nothing. An index of V or more makes the row's
    loss and gradient NaN.

    ``teacher_lse`` holds at one temperature. ``teacher_temperature``, of the
    rows' first dimension, says which: where it is not ``temperature`` the rows'
    losses are NaN, as a device cannot raise.

    ``reduction``: "mean" over the rows that count, "sum", or "none" (a loss
    per row). The record is a constant of the loss."""
    check_logits(logits)
    check_temperature(temperature)
    red = check_reduction(reduction)
    k = teacher_indices.shape[-1] if teacher_indices.dim() else 0
    if not 1 <= k <= MOST_K:
        raise ValueError(f"a record has between 1 and {MOST_K} entries, got {k}")
    rows = logits.shape[:-1]
    check_rows("teacher_indices", teacher_indices, logits, (*rows, k), False)
    check_rows("teacher_values", teacher_values, logits, (*rows, k), True)
    if teacher_lse is not None:
        check_rows("teacher_lse", teacher_lse, logits, rows, True)
    if teacher_temperature is not None:
        check_rows("teacher_temperature", teacher_temperature, logits, rows[:1], True)
        if teacher_lse is not None:
            same = teacher_temperature == temperature
            same = same.reshape(rows[:1] + (1,) * (len(rows) - 1))
            teacher_lse = torch.where(same, teacher_lse, float("nan"))
    if mask is not None:
        check_mask(mask, logits, rows)
    if logits.is_cuda:
        if teacher_values.dtype == torch.float64:
            teacher_values = teacher_values.float()
        x = kernel_rows(logits)
        loss = hip_ops().lm_distill_loss(
            x, fold(teacher_values, x, 1), fold(teacher_indices, x, 1),
            fold(teacher_lse, x), temperature, fold(mask, x), red)
        return loss.reshape(rows) if reduction == "none" else loss
    return _distill_reference(logits, teacher_values, teacher_indices,
                              teacher_lse, temperature, mask, reduction)


def _distill_reference(logits, values, indices, lse, t, mask, reduction):
    V = logits.shape[-1]
    indices = indices.long()
    present = indices >= 0
    v = values.double() / t
    some = present & ~(v == float("-inf"))
    live = some.any(-1)
    if mask is not None:
        live = live & mask
    # rows that do not count are computed on zeros, so that nothing of theirs
    # comes back through a gradient
    on = live[..., None]
    x = torch.where(on, logits, 0).to(reference_dtype(logits))
    top = x.detach().amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min)
    at = indices.clamp(0, V - 1)
    inside = torch.zeros(logits.shape, dtype=torch.int32, device=logits.device)
    inside = inside.scatter_add(-1, at, (present & (indices < V)).int()) > 0
    # subtracted before the division, and single places in 64 bits: the type's
    # lowest value stays a number
    log_s = torch.logsumexp((x - top) / t, -1, keepdim=True).double()
    log_q = (x.gather(-1, at).double() - top.double()) / t - log_s
    v = v.masked_fill(~some, float("-inf")).masked_fill(~on, 0.0)
    log_p = v - (torch.logsumexp(v, -1, keepdim=True) if lse is None
                 else lse.double()[..., None])
    p = torch.where(some, log_p.exp(), 0.0)
    use = p != 0
    rows = torch.where(use, p * (torch.where(use, log_p, 0.0)
                                 - torch.where(use, log_q, 0.0)), 0.0).sum(-1)
    if lse is not None:
        rest = (1.0 - p.sum(-1)).clamp_min(0.0)
        out = x.masked_fill(inside, float("-inf"))
        any_out = (out > float("-inf")).any(-1) | out.isnan().any(-1)
        out = torch.where(any_out[..., None], out, 0.0)
        # by a maximum of its own: far below the record its shares still differ
        low = out.detach().amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min)
        log_out = torch.logsumexp((out - low) / t, -1).double() + (
            (low.double() - top.double()) / t)[..., 0]
        rows = rows + torch.where(any_out, torch.xlogy(rest, rest)
                                  - rest * (log_out - log_s[..., 0]), 0.0)
    rows = rows * torch.where((some & (indices >= V)).any(-1), float("nan"), 1.0)
    rows = torch.where(live, rows, 0.0) * (t * t)
    loss = reduce_rows(rows, live, reduction)
    return loss if logits.dtype == torch.float64 else loss.float()
