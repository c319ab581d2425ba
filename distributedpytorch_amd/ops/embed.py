"""Token embedding with a scale, its gradient by sorted tokens.

``embedding`` (``tfm.py``) adds GPT-2's learned positions and sums the gradient with atomics; this is the lookup alone, for
models that place tokens by rotation or bias, with a gradient that is the same bit for bit in every run.
Kernels: ``csrc/embed.hip``.  Not in the reference.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _ext
from . import sink as _sink


class _SinkEmbeddingFn(torch.autograd.Function):
    """The node for a weight with a gradient sink: backward adds into the sink's buffer and reports the parameter."""

    @staticmethod
    def forward(ctx, tokens, weight, weight_lp, scale):
        ctx.save_for_backward(tokens)
        ctx.weight, ctx.scale = weight, scale
        return _ext.load().token_embedding_fwd(tokens, weight_lp, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        weight = ctx.weight
        acc = _sink.target(weight)
        dw = _ext.load().token_embedding_bwd(tokens, dy, weight.shape[0], ctx.scale, None if acc is None else acc.view(weight.shape))
        if acc is not None:
            _sink.ready(weight)
            dw = None
        return None, dw, None, None


def token_embedding(tokens: torch.Tensor, weight: torch.Tensor, weight_lp: torch.Tensor = None, *, scale: float = 1.0) -> torch.Tensor:
    """``scale * weight[tokens]`` for ``tokens`` of any shape (int64 or int32) -> ``[..., C]``.  An id outside ``[0, V)`` (the
    padding of a batch) names no row: its output is zero and it adds to no gradient.

    On the GPU ``weight [V, C]`` is the fp32 master (``C`` a multiple of 8), ``weight_lp`` its bf16 shadow (made on the fly when
    absent), the output bf16; the gradient is fp32, added into the flat gradient buffer where a sink is installed.
    First derivatives only: without a sink a backward with ``create_graph`` is refused, into one it adds as ever.
    """
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token_embedding: tokens must be int64 or int32, got {tokens.dtype}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1 or not weight.dtype.is_floating_point:
        raise ValueError(f"token_embedding: weight must be [V, C], got {weight.dtype} {tuple(weight.shape)}")
    if tokens.device != weight.device:
        raise ValueError("token_embedding: tokens and weight must be on one device")
    scale = float(scale)
    V, C = weight.shape
    if not _ext.use_hip(weight):
        live = (tokens >= 0) & (tokens < V)
        return torch.where(live[..., None], weight[torch.where(live, tokens, 0)] * scale, 0.0)
    if weight.dtype != torch.float32:
        raise TypeError(f"token_embedding: the fp32 master on the GPU, got {weight.dtype}")
    if C % 8 or C >= 1 << 24:
        raise ValueError(f"token_embedding: {C} channels: a multiple of 8 on the GPU")
    if V >= 2 ** 30 or tokens.numel() > 2 ** 27:
        raise ValueError("token_embedding: at most 2^30 - 1 rows and 2^27 tokens")
    if weight_lp is None:
        from .conv import _lp
        weight_lp = _lp(weight, None)
    elif weight_lp.shape != weight.shape or weight_lp.dtype != torch.bfloat16 or weight_lp.device != weight.device:
        raise ValueError("token_embedding: weight_lp must be the bf16 shadow of weight")
    node = _ext.load().token_embedding if _sink.of(weight) is None else _SinkEmbeddingFn.apply
    return node(tokens.contiguous(), weight, weight_lp, scale)
