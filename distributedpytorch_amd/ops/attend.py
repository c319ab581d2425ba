"""Self-attention with score modifiers: grouped key heads, a tanh cap, a distance bias, document masks, visible prefixes.

``causal_attention`` (``tfm.py``) stays the plain causal form over a packed projection, with dropout; this is the form for
rows packed with several documents, for prompts that are seen from everywhere, and for models that cap or bias their scores.
Kernels: ``csrc/attend.hip``.  Not in the reference.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ext


def _visible(B, T, causal, documents, prefix, device):
    """``[B or 1, 1, T, T]``: which key (last axis) a query sees."""
    i = torch.arange(T, device=device)
    see = (i[None, :] <= i[:, None])[None] if causal else torch.ones(1, T, T, dtype=torch.bool, device=device)
    if causal and prefix is not None:
        see = see | (i[None, None, :] < prefix[:, None, None])
    if documents is not None:
        see = see & (documents[:, :, None] == documents[:, None, :]) & (documents >= 0)[:, :, None]
    return see[:, None]


def _plain(q, k, v, causal, scale, softcap, slopes, documents, prefix):
    B, T, Hq, _ = q.shape
    group = Hq // k.shape[2]
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    if documents is not None:                      # a padded row's content reaches nothing
        pad = (documents < 0)[:, :, None, None]
        q, k, v = (t.masked_fill(pad, 0.0) for t in (q, k, v))
    qh = q.to(wide).transpose(1, 2)
    kh, vh = (t.to(wide).transpose(1, 2).repeat_interleave(group, 1) for t in (k, v))
    x = (qh @ kh.transpose(2, 3)) * scale
    if softcap:
        x = softcap * torch.tanh(x / softcap)
    if slopes is not None:
        i = torch.arange(T, device=q.device)
        x = x - slopes.to(wide)[:, None, None] * (i[:, None] - i[None, :]).abs()
    x = x.masked_fill(~_visible(B, T, causal, documents, prefix, q.device), -math.inf)
    if T:
        e = torch.exp(x - x.detach().amax(3, keepdim=True).clamp(min=-1e30))
        x = e / e.sum(3, keepdim=True).clamp(min=1e-30)
    return (x @ vh).transpose(1, 2).to(q.dtype)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True, scale: Optional[float] = None,
              softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, documents: Optional[torch.Tensor] = None,
              prefix: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Self-attention of ``q [B,T,Hq,D]`` over ``k``, ``v [B,T,Hkv,D]`` (``Hq`` a multiple of ``Hkv``; query head ``h`` reads key
    head ``h * Hkv // Hq``) -> ``[B,T,Hq,D]``.  Any strides; views of a packed projection whose rows lie on 16 bytes are read
    in place.  On the GPU: bf16, ``D`` a multiple of 8 up to 128.

    Score of query ``i`` and key ``j``: ``x = scale * q_i . k_j`` (``scale`` defaults to ``D ** -0.5``), then
    ``softcap * tanh(x / softcap)`` if ``softcap`` is not 0 (from 1e-12 to 1e12), then ``x - slopes[h] * |i - j|`` (``slopes [Hq]``, fp32).
    Visible: ``j <= i``, or ``j < prefix[b]`` (``prefix [B]``, int32, clamped to ``0 .. T``), or every ``j`` with
    ``causal=False``; and, with ``documents [B,T]`` (int32, any numbering, sorted ones run fastest), only keys of the query's
    own document.  A token with a negative document number is padding: it sees nothing, is seen by nothing, its output and
    gradients are zero, and what its rows hold does not matter.
    Rows that are not padding hold finite numbers: as in any product with probabilities of zero, a NaN or infinity there may
    reach queries that do not see it.

    Scores are formed in fp32 and lie within 1e29 of zero; past some 1e4 their own last place shows in the probabilities.
    Head dimensions up to 64 run in kernels of width 64 and the others in kernels of width 128: the products of the channels that
    are not there are computed, so 32, 80 or 96 cost what 64 or 128 do.

    Gradients for ``q``, ``k``, ``v``; the rest are constants.  Sums, statistics and scores are fp32; probabilities and
    score gradients are rounded to bf16 for the matrix products that follow them, outputs and gradients once at the end.
    Results do not depend on launch order.  On the GPU first derivatives only: a backward with ``create_graph`` is refused.
    """
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("attention: q, k, v must be [B, T, heads, D]")
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    if k.shape != v.shape or k.shape[0] != B or k.shape[1] != T or k.shape[3] != D:
        raise ValueError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not belong together")
    if Hq < 1 or Hkv < 1 or Hq % Hkv or D < 1:
        raise ValueError(f"attention: {Hq} query heads over {Hkv} key heads of {D} channels")
    if not (q.dtype == k.dtype == v.dtype and q.dtype.is_floating_point):
        raise TypeError("attention: q, k, v must share one floating type")
    if not q.device == k.device == v.device:
        raise ValueError("attention: q, k, v must be on one device")
    scale = D ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not 1e-12 < scale < 1e12:
        raise ValueError(f"attention: scale must be positive and finite, got {scale}")
    if softcap != 0.0 and not 1e-12 < softcap < 1e12:
        raise ValueError(f"attention: softcap must be 0 (none) or between 1e-12 and 1e12, got {softcap}")
    for name, t, shape, dtype in (("slopes", slopes, (Hq,), torch.float32), ("documents", documents, (B, T), torch.int32),
                                  ("prefix", prefix, (B,), torch.int32)):
        if t is None:
            continue
        if t.shape != shape or t.dtype != dtype:
            raise ValueError(f"attention: {name} must be {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
        if t.device != q.device:
            raise ValueError(f"attention: {name} must be on q's device")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"attention: {name} gets no gradient")
    if not _ext.use_hip(q):
        return _plain(q, k, v, causal, scale, softcap, slopes, documents, prefix)
    if q.dtype != torch.bfloat16:
        raise TypeError(f"attention: bf16 on the GPU, got {q.dtype}")
    if D % 8 or D > 128:
        raise ValueError(f"attention: head dimension {D}: a multiple of 8 up to 128 on the GPU")
    if B > 65535 or Hq > 65535 or Hq * D >= 1 << 23 or T > 1 << 22:
        raise ValueError("attention: at most 65,535 rows, 65,535 heads, 2^23 - 1 channels and 2^22 tokens in a row")
    slopes, documents, prefix = (t if t is None else t.contiguous() for t in (slopes, documents, prefix))
    return _ext.load().attention_ex(q, k, v, bool(causal), scale, softcap, slopes, documents, prefix)
