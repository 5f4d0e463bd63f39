"""Layer norm on the sm_100a kernels (csrc/misc/layer_norm.cu), forward and backward:

    mu = mean_j x,  rstd = 1 / sqrt(mean_j (x - mu)^2 + eps),  xhat = (x - mu) rstd,  y = xhat * weight + bias
    g = dy * weight,  dx = rstd (g - mean_j g - xhat mean_j (g xhat)),  dweight = sum_n dy xhat,  dbias = sum_n dy

``models.normalization.LayerNorm`` is the module that uses it and, in plain PyTorch, its definition.
"""
from __future__ import annotations

import torch

from ._ext import lib

MAX_DIM = 16384
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Normalise ``x`` (..., d) over its last dimension.

    ``x``: fp32, bf16 or fp16 on CUDA, any strides (rows with a unit column stride are read in place),
    1 <= d <= 16384.  ``weight`` and the optional ``bias``: fp32 [d].  The result is ``out_dtype`` (default
    x's), dense.  Statistics and sums are fp32; the result is rounded once.  Runs on the current stream.

    Differentiable with respect to ``x``, ``weight`` and ``bias``: the backward reads ``x`` again with the forward's
    per-row mean and rstd, and sums the weight and bias gradients in a fixed order (the same inputs give the same bits).
    Second derivatives and forward-mode tangents are refused (``models.normalization.LayerNorm.plain`` has them)."""
    if not x.is_cuda:
        raise ValueError("layer_norm: x must be a CUDA tensor (models.normalization.LayerNorm has the CPU form)")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if x.dtype not in _FLOATS or out_dtype not in _FLOATS:
        raise TypeError(f"layer_norm: x and the result must be float32, bfloat16 or float16, not {x.dtype} -> {out_dtype}")
    d = x.shape[-1] if x.dim() else 0
    if not 1 <= d <= MAX_DIM:
        raise ValueError(f"layer_norm: the last dimension must be between 1 and {MAX_DIM}, not {d}")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps must not be negative ({eps})")
    rows = x if x.dim() == 2 else x.reshape(-1, d)
    if d > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    y = lib().layer_norm(rows, weight.contiguous(), bias.contiguous() if bias is not None else None, eps, out_dtype)
    return y if x.dim() == 2 else y.view(x.shape)
