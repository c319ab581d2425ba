"""Distillation loss from a teacher's top logits, loss and gradient in one pass over the student's.

Kernels: ``csrc/distill.hip``.  Not in the reference.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ext

MAX_ENTRIES = 1024                       # teacher entries of a row on the GPU: one to four per thread of a workgroup


def _plain(logits, ids, teacher, n_classes, tau):
    N = max(logits.shape[0], 1)
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    z = logits[:, :n_classes].to(wide) / tau
    live = (ids >= 0) & (ids < n_classes) & (teacher != -math.inf)
    rows = live.any(1)
    z = torch.where(rows[:, None], z, 0.0)               # a row without a teacher gives nothing, whatever it holds
    z = z - z.detach().amax(1, keepdim=True)             # what all classes share would cost the rest its digits
    lse = torch.logsumexp(z, 1, keepdim=True)
    t = (teacher.to(wide) / tau).masked_fill(~live, -math.inf).masked_fill(~rows[:, None], 0.0)
    logp = torch.log_softmax(t, 1)
    p = logp.exp() * rows[:, None]
    logq = z.gather(1, torch.where(live, ids, 0).long()) - lse
    term = torch.where(live & (p != 0), p * (torch.where(live, logp, 0.0) - logq), 0.0)
    return tau * tau * term.sum() / N


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *, temperature: float = 1.0,
                      n_classes: Optional[int] = None) -> torch.Tensor:
    """``temperature^2 * KL(p || q)``, mean over ALL rows of ``logits [..., ld]`` (only the first ``n_classes`` columns are classes;
    the rest is padding), as an fp32 scalar (fp64 for fp64 logits off the GPU): ``q = softmax(logits / temperature)`` over the classes, ``p`` the softmax of the
    row's ``teacher_logits [..., K] / temperature`` over its live entries, whose classes ``teacher_ids [..., K]`` (int64 or
    int32) names.  An entry is dead when its id lies outside ``[0, n_classes)`` or its logit is ``-inf`` (short lists are
    padded so); an id may come twice; a row without live entries (a prompt's) contributes zero loss and gradient.

    Gradient for ``logits`` (its type; fp32 arithmetic, rounded once), zero in the padding columns.  ``logits`` are not changed.
    On the GPU: bf16 or fp32 logits, fp32 teacher logits, ``K`` up to 1024.  There the forward writes the gradient for an upstream
    gradient of 1, and any other (a weight beside a second loss, accumulation) costs backward another pass over the logits; first
    derivatives only: a backward with ``create_graph`` is refused.
    """
    if logits.dim() < 1 or not logits.dtype.is_floating_point:
        raise ValueError("distillation_loss: logits must be floating point [..., columns]")
    ld = logits.shape[-1]
    n_classes = ld if n_classes is None else int(n_classes)
    if not 1 <= n_classes <= ld:
        raise ValueError(f"distillation_loss: {n_classes} classes in {ld} columns")
    temperature = float(temperature)
    if not 1e-6 < temperature < 1e6:
        raise ValueError(f"distillation_loss: temperature must be positive and finite, got {temperature}")
    if teacher_ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"distillation_loss: teacher_ids must be int64 or int32, got {teacher_ids.dtype}")
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.dim() != logits.dim() or teacher_ids.shape[:-1] != logits.shape[:-1] \
            or teacher_ids.shape[-1] < 1:
        raise ValueError(f"distillation_loss: logits {tuple(logits.shape)}, teacher_ids {tuple(teacher_ids.shape)}, "
                         f"teacher_logits {tuple(teacher_logits.shape)} do not belong together")
    if not teacher_logits.dtype.is_floating_point:
        raise TypeError("distillation_loss: teacher_logits must be floating point")
    if not logits.device == teacher_ids.device == teacher_logits.device:
        raise ValueError("distillation_loss: logits and teacher must be on one device")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("distillation_loss: teacher_logits get no gradient")
    K = teacher_ids.shape[-1]
    if logits.dim() != 2:                          # (a view is a node of its own in backward: none where none is needed)
        logits, teacher_ids, teacher_logits = logits.reshape(-1, ld), teacher_ids.reshape(-1, K), teacher_logits.reshape(-1, K)
    if not _ext.use_hip(logits):
        return _plain(logits, teacher_ids, teacher_logits, n_classes, temperature)
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"distillation_loss: bf16 or fp32 logits on the GPU, got {logits.dtype}")
    if teacher_logits.dtype != torch.float32:
        raise TypeError(f"distillation_loss: fp32 teacher logits on the GPU, got {teacher_logits.dtype}")
    if K > MAX_ENTRIES:
        raise ValueError(f"distillation_loss: {K} teacher entries per row, at most {MAX_ENTRIES} on the GPU")
    if ld >= 1 << 30 or logits.shape[0] >= 1 << 31:
        raise ValueError("distillation_loss: at most 2^30 - 1 columns and 2^31 - 1 rows")
    return _ext.load().distillation_loss(logits.contiguous(), teacher_ids.contiguous(), teacher_logits.contiguous(), n_classes, temperature)
