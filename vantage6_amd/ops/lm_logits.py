"""What the losses over language-model logits share (csrc/lm_loss.hip).

Argument checks, the layout that the kernels read, and the CPU path's types
and reductions. The kernels take ``[V]``, ``[T, V]`` or ``[B, T, V]`` logits
whose rows may lie anywhere (a slice ``logits[:, :-1]`` is read in place);
more dimensions are folded into ``B``, and logits whose last dimension is
not contiguous are copied once. A call takes up to 2**22 - 1 rows.
"""
from __future__ import annotations

import torch

REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}

_KERNEL_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def check_logits(logits: torch.Tensor) -> None:
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 28:
        raise ValueError("logits must be [..., V] with 1 <= V < 2**28")
    if logits.is_cuda and logits.numel() >= logits.shape[-1] << 22:
        raise ValueError("logits must be of fewer than 2**22 rows a call")
    if logits.dtype not in _KERNEL_TYPES and (
            logits.is_cuda or logits.dtype != torch.float64):
        raise ValueError("logits must be bfloat16, float16 or float32 "
                         f"(float64 on the CPU alone), got {logits.dtype}")


def check_rows(name: str, t: torch.Tensor, logits: torch.Tensor, want,
               floating: bool | None = None) -> None:
    """``t`` has the shape ``want`` (the rows' or more), on the logits' device;
    of floats, or (``floating`` False) of int64 or int32."""
    if t.shape != want:
        raise ValueError(f"{name} must have shape {tuple(want)}, got {tuple(t.shape)}")
    if t.device != logits.device:
        raise ValueError(f"{name} is on {t.device}, logits on {logits.device}")
    if floating:
        if not t.is_floating_point():
            raise ValueError(f"{name} must be floating point, got {t.dtype}")
        if t.requires_grad and torch.is_grad_enabled():
            # not to drop a gradient that the caller may expect
            raise ValueError(f"{name} is a constant of this loss: detach it")
    elif floating is False and t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32, got {t.dtype}")


def check_mask(mask: torch.Tensor, logits: torch.Tensor, want) -> None:
    if mask.dtype != torch.bool:
        raise ValueError(f"mask must be bool, got {mask.dtype}")
    check_rows("mask", mask, logits, want)


def check_reduction(reduction: str) -> int:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(REDUCTIONS)}, "
                         f"got {reduction!r}")
    return REDUCTIONS[reduction]


def check_temperature(temperature: float) -> None:
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError("temperature must be between 1e-3 and 1e3, "
                         f"got {temperature}")


def kernel_rows(logits: torch.Tensor) -> torch.Tensor:
    """``logits`` as the kernels read them: at most 3-D, rows contiguous."""
    if logits.dim() > 3:
        logits = logits.flatten(0, -3)
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    return logits


def fold(t: torch.Tensor | None, x: torch.Tensor, more: int = 0
         ) -> torch.Tensor | None:
    """A per-row tensor (with ``more`` dimensions of its own behind the rows')
    in the row shape of ``x = kernel_rows(logits)``."""
    if t is None or t.dim() - more == x.dim() - 1:
        return t
    return t.reshape(*x.shape[:-1], *t.shape[t.dim() - more:])


def reference_dtype(t: torch.Tensor) -> torch.dtype:
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def reduce_rows(rows: torch.Tensor, live: torch.Tensor | None,
                reduction: str) -> torch.Tensor:
    """Mean over the rows that count (0 if none does), sum, or the rows."""
    if reduction == "none":
        return rows
    if reduction == "sum":
        return rows.sum()
    n = rows.numel() if live is None else live.sum().clamp_min(1)
    return rows.sum() / max(n, 1) if live is None else rows.sum() / n
