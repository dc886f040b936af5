"""Layer norm over the last axis, on sm_100a kernels (``fdwt_layer_norm_forward`` and
``fdwt_layer_norm_backward`` in ``include/fdwt_b200.h``).

    y = (x - mean x) / sqrt(mean (x - mean x)^2 + eps) * weight + bias

The reference's token mixers come without a norm; a block around them needs one before the
mixer.  Inputs must be CUDA tensors, fp32, fp64, fp16 or bf16; statistics and sums are fp32 (fp64
for fp64 inputs).
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["layer_norm", "LayerNorm"]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, eps: float, codes, want_stats: bool):
    shape = x.shape
    dim = shape[-1]
    rows = x.numel() // dim
    dev = x.device
    y = torch.empty_like(x)
    stats = None
    if want_stats:
        stats = torch.empty((rows, 2), device=dev,
                            dtype=torch.float64 if codes[0] == 1 else torch.float32)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_layer_norm_forward(
            codes[0], codes[1], rows, dim, x.data_ptr(), _ptr(weight), _ptr(bias), eps,
            y.data_ptr(), _ptr(stats), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_layer_norm_forward")
    return y, stats


@lru_cache(maxsize=1024)
def _backward_ws(code: int, rows: int, dim: int, need_params: int, device_index: int) -> int:
    """Workspace bytes of a backward call (a pure function of its sizes on one device)."""
    return int(_lib.load().fdwt_layer_norm_backward_workspace(code, rows, dim, need_params))


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
        need_x, need_w, need_b, _, _ = ctx.needs_input_grad
        code, param = ctx.codes
        dy = dy.contiguous()
        dim = x.shape[-1]
        rows = x.numel() // dim
        dev = x.device
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty(dim, device=dev, dtype=_lib.DTYPE_OF[param]) if need_w else None
        db = torch.empty(dim, device=dev, dtype=_lib.DTYPE_OF[param]) if need_b else None
        with _lib.device_guard(dev):
            nws = _backward_ws(code, rows, dim, int(need_w or need_b), dev.index)
            ws = _lib.workspace(nws, dev)
            st = _lib.load().fdwt_layer_norm_backward(
                code, param, rows, dim, dy.data_ptr(), x.data_ptr(), _ptr(weight),
                stats.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nws,
                _lib.raw_stream(dev.index))
        if st:
            _lib.check(st, "fdwt_layer_norm_backward")
        return dx, dw, db, None, None


def _parameter(name: str, p: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    if p.shape != x.shape[-1:]:
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
    if p.dtype != x.dtype and (p.dtype != torch.float32 or x.dtype == torch.float64):
        raise TypeError(f"{name} must be {x.dtype} or torch.float32 "
                        f"(torch.float64 for float64 inputs), got {p.dtype}")
    return p.contiguous()


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
    x = x.contiguous()
    param, needs = code, x.requires_grad
    if weight is not None:
        weight = _parameter("weight", weight, x)
        param, needs = _lib.DTYPES[weight.dtype], needs or weight.requires_grad
    if bias is not None:
        bias = _parameter("bias", bias, x)
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError(f"weight and bias must have one type, got {weight.dtype} and "
                            f"{bias.dtype}")
        param, needs = _lib.DTYPES[bias.dtype], needs or bias.requires_grad
    if (needs and torch.is_grad_enabled()) or _lib.has_tangent(x, weight, bias):
        return _LayerNormFunction.apply(x, weight, bias, float(eps), (code, param))
    return _forward(x, weight, bias, float(eps), (code, param), False)[0]


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
