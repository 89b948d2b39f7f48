"""Model + loss factory used by the fedavg algorithm packages and bench."""
from __future__ import annotations

from typing import Callable

import torch
import torch.nn.functional as F


def build_model(name: str, device="cpu", dtype=torch.bfloat16, **kw) -> torch.nn.Module:
    name = name.lower()
    if name in ("logreg", "logistic_regression"):
        from .logreg import logreg

        return logreg(device=device, dtype=dtype, **kw)
    if name in ("resnet18", "resnet-18"):
        from .resnet import resnet18

        return resnet18(device=device, dtype=dtype, **kw)
    if name in ("resnet50", "resnet-50"):
        from .resnet import resnet50

        return resnet50(device=device, dtype=dtype, **kw)
    if name in ("bert", "bert_base", "bert-base"):
        from .transformer import bert_base

        return bert_base(device=device, dtype=dtype, **kw)
    if name in ("llama", "llama_1b", "llama-1b", "llama-3-1b"):
        from .transformer import llama_1b

        return llama_1b(device=device, dtype=dtype, **kw)
    if name in ("vit", "vit_b16", "vit-b16"):
        from .transformer import vit_b16

        return vit_b16(device=device, dtype=dtype, **kw)
    raise ValueError(f"unknown model {name!r}")


_LM_NAMES = ("bert", "bert_base", "bert-base", "llama", "llama_1b", "llama-1b",
             "llama-3-1b")


def _lm_logits(model, ids):
    """Logits over the real vocabulary: a padded head's extra columns are cut
    off as a view, which the losses over logits read in place."""
    logits = model(ids)
    vl = getattr(model, "vocab_logical", logits.shape[-1])
    return logits[..., :vl] if vl < logits.shape[-1] else logits


def _distill_objective(options) -> Callable:
    """Batch: ``input_ids`` [N, S] and the teacher's record of every position,
    ``teacher_values`` and ``teacher_indices`` [N, S, k], optionally
    ``teacher_lse`` and ``mask`` [N, S], and ``teacher_temperature`` [N]."""
    def loss(model, batch):
        from ..ops.distill import distill_loss

        return distill_loss(
            _lm_logits(model, batch["input_ids"]), batch["teacher_values"],
            batch["teacher_indices"], batch.get("teacher_lse"), mask=batch.get("mask"),
            teacher_temperature=batch.get("teacher_temperature"), **options)

    return loss


def _preference_objective(options) -> Callable:
    """Batch: ``input_ids`` [N, 2, S] (chosen, rejected), ``ref_logps`` [N, 2],
    optionally ``mask`` [N, 2, S], True where a token is one of the answer."""
    ignore = options.get("ignore_index", -100)

    def loss(model, batch):
        from ..ops.preference import preference_loss

        ids = batch["input_ids"].transpose(0, 1).flatten(0, 1)
        targets = ids[:, 1:]
        if "mask" in batch:
            mask = batch["mask"].transpose(0, 1).flatten(0, 1)[:, 1:]
            targets = torch.where(mask, targets, ignore)
        ref = batch["ref_logps"].transpose(0, 1).flatten()
        return preference_loss(_lm_logits(model, ids[:, :-1]), targets, ref,
                               **options).loss

    return loss


def _policy_objective(options) -> Callable:
    """Batch: ``input_ids`` [N, S]; of the tokens that its positions 1.. hold,
    ``old_logps``, ``advantages`` and optionally ``ref_logps`` [N, S - 1];
    optionally ``mask`` [N, S], True where a token was sampled."""
    def loss(model, batch):
        from ..ops.preference import policy_loss

        ids = batch["input_ids"]
        mask = batch["mask"][:, 1:] if "mask" in batch else None
        return policy_loss(_lm_logits(model, ids[:, :-1]), ids[:, 1:],
                           batch["old_logps"], batch["advantages"],
                           batch.get("ref_logps"), mask=mask, **options).loss

    return loss


_OBJECTIVES = {"distill": _distill_objective, "preference": _preference_objective,
               "policy": _policy_objective}


@torch.no_grad()
def teacher_record(model, input_ids, k: int = 64, temperature: float = 1.0) -> dict:
    """What a station publishes of its model's answers to ``input_ids``: the
    entries that the "distill" objective's batches hold. ``teacher_lse`` is of
    ``temperature``, the objective's own; ``teacher_temperature`` [N] says so."""
    from ..ops.distill import topk_logits

    top = topk_logits(_lm_logits(model, input_ids), k, temperature)
    return {"teacher_values": top.values, "teacher_indices": top.indices,
            "teacher_lse": top.logsumexp,
            "teacher_temperature": torch.full(
                input_ids.shape[:1], float(temperature), dtype=torch.float64,
                device=top.values.device)}


def model_loss(name: str, objective: str | None = None, **options) -> Callable:
    """(model, batch) -> scalar loss, fp32 loss computation.

    Language models take an ``objective`` other than the next token:
    "distill", "preference" or "policy", with ``options`` for its loss
    (``temperature``, ``beta``, ``kl_coef``, ...)."""
    name = name.lower()
    if objective is not None:
        if name not in _LM_NAMES or objective not in _OBJECTIVES:
            raise ValueError(f"no objective {objective!r} for model {name!r}")
        return _OBJECTIVES[objective](options)
    if options:
        raise ValueError(f"options {sorted(options)} need an objective")
    if name in _LM_NAMES:

        def lm_loss(model, batch):
            from ..ops.cross_entropy import cross_entropy

            ids = batch["input_ids"]
            logits = model(ids[:, :-1])
            vl = getattr(model, "vocab_logical", logits.shape[-1])
            if vl < logits.shape[-1]:
                # padded LM head (BertBase vocab_pad): pad classes get
                # probability exactly 0 and exactly-zero grads
                logits = logits.clone()
                logits[..., vl:] = float("-inf")
            return cross_entropy(logits, ids[:, 1:])

        return lm_loss

    def cls_loss(model, batch):
        logits = model(batch["x"])
        return F.cross_entropy(logits.float(), batch["y"])

    return cls_loss


def model_loss_per_sample(name: str) -> Callable:
    """(model, batch) -> per-sample loss vector [B] (DP-SGD needs this)."""
    name = name.lower()
    if name in _LM_NAMES:

        def lm_loss_ps(model, batch):
            from ..ops.cross_entropy import cross_entropy

            ids = batch["input_ids"]
            logits = model(ids[:, :-1])
            losses = cross_entropy(logits, ids[:, 1:], reduction="none")
            return losses.reshape(ids.shape[0], -1).mean(-1)

        return lm_loss_ps

    def cls_loss_ps(model, batch):
        logits = model(batch["x"])
        return F.cross_entropy(logits.float(), batch["y"], reduction="none")

    return cls_loss_ps
