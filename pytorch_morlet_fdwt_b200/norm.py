"""Layer norm over the last axis, on sm_100a kernels (``fdwt_layer_norm_forward`` and
``fdwt_layer_norm_backward`` in ``include/fdwt_b200.h``).

    y = (x - mean x) / sqrt(mean (x - mean x)^2 + eps) * weight + bias

The reference's token mixers come without a norm; a block around them needs one before the
mixer.  Inputs must be CUDA tensors, fp32, fp64, fp16 or bf16; statistics and sums are fp32 (fp64
for fp64 inputs).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["layer_norm", "LayerNorm"]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, eps: float, codes, want_stats: bool):
    dim = x.shape[-1]
    rows = x.numel() // dim
    dev = x.device
    y = torch.empty_like(x)
    stats = None
    if want_stats:
        acc = torch.float64 if x.dtype == torch.float64 else torch.float32
        stats = torch.empty((rows, 2), device=dev, dtype=acc)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_layer_norm_forward(
            codes[0], codes[1], rows, dim, x.data_ptr(), _ptr(weight), _ptr(bias), eps,
            y.data_ptr(), _ptr(stats), _lib.stream_of(dev))
    _lib.check(st, "fdwt_layer_norm_forward")
    return y, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps: float, codes):
        y, stats = _forward(x, weight, bias, eps, codes, True)
        ctx.codes = codes
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy = dy.contiguous()
        dim = x.shape[-1]
        rows = x.numel() // dim
        dev = x.device
        param = _lib.DTYPE_OF[ctx.codes[1]]
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty(dim, device=dev, dtype=param) if need_w else None
        db = torch.empty(dim, device=dev, dtype=param) if need_b else None
        lib = _lib.load()
        with _lib.device_guard(dev):
            nws = lib.fdwt_layer_norm_backward_workspace(ctx.codes[0], rows, dim,
                                                         int(need_w or need_b))
            ws = _lib.workspace(nws, dev)
            st = lib.fdwt_layer_norm_backward(
                ctx.codes[0], ctx.codes[1], rows, dim, dy.data_ptr(), x.data_ptr(), _ptr(weight),
                stats.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nws,
                _lib.stream_of(dev))
        _lib.check(st, "fdwt_layer_norm_backward")
        return dx, dw, db, None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of ``x (..., D)`` over its last axis; ``weight`` and ``bias`` are ``(D,)`` (or
    None), both of x's type or both fp32.  Differentiable once in x, weight and bias; the
    gradients' sums over rows are added in a fixed order."""
    _lib.require_cuda(x, weight, bias)
    code = _lib.dtype_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected (..., D) with D >= 1, got shape {tuple(x.shape)}")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    param = code
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != x.shape[-1:]:
            raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.dtype != x.dtype and (p.dtype != torch.float32 or x.dtype == torch.float64):
            raise TypeError(f"{name} must be {x.dtype} or torch.float32 "
                            f"(torch.float64 for float64 inputs), got {p.dtype}")
        param = _lib.dtype_code(p.dtype)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    codes = (code, param)
    if torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad)
            or (bias is not None and bias.requires_grad)):
        return _LayerNormFunction.apply(x, weight, bias, float(eps), codes)
    return _forward(x, weight, bias, float(eps), codes, False)[0]


class LayerNorm(nn.Module):
    """:func:`layer_norm` with learned ``weight`` (ones) and ``bias`` (zeros) of ``(dim,)``."""

    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, eps={self.eps}"
