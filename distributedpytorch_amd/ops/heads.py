"""Norms of query and key heads with the position rotation in the same pass, over the packed projection.

Kernels: ``csrc/heads.hip``.  Not in the reference.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _ext


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """``theta ** (-2 i / rotary_dim)`` for ``i < rotary_dim / 2``, fp64: made once and kept beside the model."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim must be even and positive, got {rotary_dim}")
    return float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)


def _plain(qkv, n_head, n_kv_head, q_weight, k_weight, inv_freq, positions, eps, interleaved):
    B, T, C = qkv.shape
    n = n_head + 2 * n_kv_head
    x = qkv.reshape(B, T, n, C // n)
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32

    def one(h, w):
        h = h.to(wide)
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(3, keepdim=True) + eps) * w.to(wide)
        if inv_freq is not None:
            R = 2 * inv_freq.numel()
            at = torch.arange(T, device=x.device).expand(B, T) if positions is None else positions
            angle = (at.double()[..., None] * inv_freq)[:, :, None]
            cos, sin = angle.cos().to(wide), angle.sin().to(wide)
            r, rest = h[..., :R], h[..., R:]
            a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, 3)
            a, b = a * cos - b * sin, b * cos + a * sin
            h = torch.cat((torch.stack((a, b), 4).flatten(3) if interleaved else torch.cat((a, b), 3), rest), 3)
        return h.to(x.dtype)

    return one(x[:, :, :n_head], q_weight), one(x[:, :, n_head:n_head + n_kv_head], k_weight), x[:, :, n_head + n_kv_head:]


def qk_norm_rotary(qkv: torch.Tensor, n_head: int, n_kv_head: Optional[int] = None, *, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                   positions: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``qkv [B, T, (n_head + 2 n_kv_head) * D]`` (q | k | v along the last axis, heads contiguous inside each, as
    ``causal_attention`` takes it) -> ``q [B,T,n_head,D]``, ``k`` and ``v [B,T,n_kv_head,D]`` for ``attention``.

    ``q_weight``, ``k_weight`` (both ``[D]``, fp32, or neither): each query and key head is divided by its root mean square
    (``eps`` inside the root) and multiplied by the gain, which all heads share.  ``inv_freq`` (``[R/2]``, fp64,
    ``rotary_frequencies``): the first ``R`` channels are rotated in pairs by ``positions[b, t] * inv_freq[i]``, pairs being
    ``(i, i + R/2)``, or ``(2i, 2i + 1)`` with ``interleaved``; ``positions`` (int64, ``[T]`` or ``[B,T]``, default
    ``0 .. T-1``) may be any whole numbers, angles are formed in 64 bits.  On the GPU: bf16, ``D`` a multiple of 8 up to 256,
    ``R`` a multiple of 16.  ``v`` is a view of ``qkv``.

    Gradients for ``qkv`` and the two gains (fp32, summed in a fixed order); on the GPU first derivatives only: a backward with
    ``create_graph`` is refused.
    """
    n_kv_head = n_head if n_kv_head is None else n_kv_head
    if qkv.dim() != 3 or n_head < 1 or n_kv_head < 1 or qkv.shape[2] == 0 or qkv.shape[2] % (n_head + 2 * n_kv_head):
        raise ValueError(f"qk_norm_rotary: qkv {tuple(qkv.shape)} does not hold {n_head} + 2 x {n_kv_head} heads")
    B, T, C = qkv.shape
    D = C // (n_head + 2 * n_kv_head)
    if not qkv.dtype.is_floating_point:
        raise TypeError("qk_norm_rotary: qkv must be floating point")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("qk_norm_rotary: q_weight and k_weight go together")
    if q_weight is None and inv_freq is None:
        raise ValueError("qk_norm_rotary: neither gains nor frequencies given")
    if positions is not None and inv_freq is None:
        raise ValueError("qk_norm_rotary: positions without frequencies")
    if not (eps >= 0.0 and eps < 1e30):
        raise ValueError(f"qk_norm_rotary: eps must not be negative, got {eps}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (D,) or not w.dtype.is_floating_point or w.device != qkv.device):
            raise ValueError(f"qk_norm_rotary: {name} must be [{D}] on qkv's device")
    if inv_freq is not None:
        if inv_freq.dim() != 1 or inv_freq.dtype != torch.float64 or inv_freq.device != qkv.device or not 2 <= 2 * inv_freq.numel() <= D:
            raise ValueError(f"qk_norm_rotary: inv_freq must be fp64 [R / 2] with 2 <= R <= {D}, on qkv's device")
        if inv_freq.requires_grad and torch.is_grad_enabled():
            raise ValueError("qk_norm_rotary: inv_freq gets no gradient")
    if positions is not None:
        if positions.dtype != torch.int64 or positions.shape not in ((T,), (B, T)) or positions.device != qkv.device:
            raise ValueError("qk_norm_rotary: positions must be int64 [T] or [B, T] on qkv's device")
        positions = positions.expand(B, T)
    if not _ext.use_hip(qkv):
        return _plain(qkv, n_head, n_kv_head, q_weight, k_weight, inv_freq, positions, eps, interleaved)
    if qkv.dtype != torch.bfloat16 or (q_weight is not None and not q_weight.dtype == k_weight.dtype == torch.float32):
        raise TypeError("qk_norm_rotary: bf16 qkv and fp32 gains on the GPU")
    if D % 8 or D > 256:
        raise ValueError(f"qk_norm_rotary: head dimension {D}: a multiple of 8 up to 256 on the GPU")
    if inv_freq is not None and inv_freq.numel() % 8:
        raise ValueError(f"qk_norm_rotary: {2 * inv_freq.numel()} rotated channels: a multiple of 16 on the GPU")
    if not qkv.is_contiguous():
        qkv = qkv.contiguous()
    q_weight, k_weight, inv_freq, positions = (t if t is None else t.contiguous() for t in (q_weight, k_weight, inv_freq, positions))
    return tuple(_ext.load().qk_norm_rotary(qkv, q_weight, k_weight, inv_freq, positions, n_head, n_kv_head, float(eps), bool(interleaved)))
