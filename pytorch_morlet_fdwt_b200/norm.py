"""Norms over the last axis, on sm_100a kernels (``fdwt_layer_norm_*`` and ``fdwt_rms_norm_*`` in
``include/fdwt_b200.h``).

    layer norm    y = (x - mean x) / sqrt(mean (x - mean x)^2 + eps) * weight + bias
    rms norm      total = x + residual,  y = total / sqrt(mean total^2 + eps) * weight

The reference's token mixers come without a norm; a block around them needs one before the
mixer, and a stack of blocks the residual's addition with it.  Inputs must be CUDA tensors, fp32,
fp64, fp16 or bf16; statistics and sums are fp32 (fp64 for fp64 inputs).
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple, Union

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["layer_norm", "LayerNorm", "rms_norm", "rms_norm_quantized", "RMSNorm"]

# codes of fdwt_rms_norm_quantized
_QUANTIZED = {torch.float8_e4m3fn: 0, torch.int8: 1}


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


# ------------------------------------------------------------------------------ rms norm


def _rms_forward(x, residual, weight, eps: float, codes, want_rstd: bool):
    dim = x.shape[-1]
    rows = x.numel() // dim
    dev = x.device
    y = torch.empty_like(x)
    total = None if residual is None else torch.empty_like(residual)
    rstd = None
    if want_rstd:
        rstd = x.new_empty(rows, dtype=torch.float64 if codes[0] == 1 else torch.float32)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_rms_norm_forward(
            *codes, rows, dim, x.data_ptr(), _ptr(residual), _ptr(weight), eps, y.data_ptr(),
            _ptr(total), _ptr(rstd), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_rms_norm_forward")
    return y, total, rstd


@lru_cache(maxsize=1024)
def _rms_backward_ws(code: int, rows: int, dim: int, need_weight: int, device_index: int) -> int:
    """Workspace bytes of a backward call (a pure function of its sizes on one device)."""
    return int(_lib.load().fdwt_rms_norm_backward_workspace(code, rows, dim, need_weight))


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps: float, codes):
        y, total, rstd = _rms_forward(x, residual, weight, eps, codes, True)
        ctx.set_materialize_grads(False)
        ctx.codes, ctx.added = codes, residual is not None
        ctx.save_for_backward(x if total is None else total, weight, rstd)
        return y if total is None else (y, total)

    @staticmethod
    @_lib.once
    def backward(ctx, dy, dtotal=None):
        total, weight, rstd = ctx.saved_tensors
        need_x, need_r, need_w, _, _ = ctx.needs_input_grad
        code, stream_code, param = ctx.codes
        if dy is None and dtotal is None:
            return (None,) * 5
        dtype = _lib.DTYPE_OF[code]
        if dy is None:  # the sum alone was used
            dw = torch.zeros_like(weight) if need_w else None
            return dtotal.to(dtype), dtotal if ctx.added else None, dw, None, None
        dy = dy.contiguous()
        if dtotal is not None:
            dtotal = dtotal.contiguous()
        dim = total.shape[-1]
        rows = total.numel() // dim
        dev = total.device
        need = need_x or need_r
        dx = torch.empty_like(dy) if need else None
        dr = torch.empty_like(total) if need_r and stream_code != code else None
        dw = torch.empty_like(weight) if need_w else None
        with _lib.device_guard(dev):
            nws = _rms_backward_ws(code, rows, dim, int(need_w), dev.index)
            ws = _lib.workspace(nws, dev)
            st = _lib.load().fdwt_rms_norm_backward(
                code, stream_code, param, rows, dim, dy.data_ptr(), _ptr(dtotal),
                total.data_ptr(), _ptr(weight), rstd.data_ptr(), _ptr(dx), _ptr(dr), _ptr(dw),
                _ptr(ws), nws, _lib.raw_stream(dev.index))
        if st:
            _lib.check(st, "fdwt_rms_norm_backward")
        if stream_code == code:
            dr = dx
        return dx, dr if need_r else None, dw, None, None


def _rms_inputs(x, weight, residual, eps: float):
    """The checked inputs of a call, contiguous, with their type codes."""
    _lib.require_cuda(x, weight, residual)
    code = param = stream = _lib.dtype_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"expected (..., D) with D >= 1, got shape {tuple(x.shape)}")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    x = x.contiguous()
    if weight is not None:
        weight = _parameter("weight", weight, x)
        param = _lib.DTYPES[weight.dtype]
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got "
                             f"{tuple(residual.shape)}")
        if residual.dtype != x.dtype and (residual.dtype != torch.float32
                                          or x.dtype == torch.float64):
            raise TypeError(f"residual must be {x.dtype} or torch.float32 (torch.float64 for "
                            f"float64 inputs), got {residual.dtype}")
        residual = residual.contiguous()
        stream = _lib.DTYPES[residual.dtype]
    return x, weight, residual, (code, stream, param)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
             residual: Optional[torch.Tensor] = None, eps: float = 1e-6
             ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Root-mean-square norm of ``x (..., D)`` over its last axis, or, with a ``residual`` of x's
    shape, of ``total = x + residual``: then ``(y, total)`` is returned, for the next residual.

    ``weight (D,)`` (or None) and ``residual`` are of x's type or fp32; total has the residual's
    type and is rounded to it before the norm, so that the result is that of an addition and a
    norm of its result.  Differentiable once in x, weight and residual; the gradients' sums over
    rows are added in a fixed order."""
    x, weight, residual, codes = _rms_inputs(x, weight, residual, eps)
    if _lib.needs_grad(x, weight, residual) or _lib.has_tangent(x, weight, residual):
        return _RMSNormFunction.apply(x, residual, weight, float(eps), codes)
    y, total, _ = _rms_forward(x, residual, weight, float(eps), codes, False)
    return y if total is None else (y, total)


def rms_norm_quantized(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                       residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       group_size: Optional[int] = None,
                       dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[torch.Tensor, ...]:
    """:func:`rms_norm` with its result in 8 bits: ``(q, scales)``, or ``(q, scales, total)`` with
    a residual; ``q (..., D)`` of ``dtype`` (``torch.float8_e4m3fn`` or ``torch.int8``) and fp32
    ``scales (..., D // group_size)``, so that ``q * scale`` is the result.

    Groups of ``group_size`` neighbouring values (a divisor of D; the whole row by default) share
    a scale, their largest magnitude over 448 (e4m3) or 127 (int8), at least ``2 ** -126``, and 1
    where all are zero; the result is formed in 32 bits and rounded once, to 8.  A NaN makes its
    group's scale NaN.  For fp32, fp16 and bf16 inputs.  No gradient."""
    x, weight, residual, codes = _rms_inputs(x, weight, residual, eps)
    if dtype not in _QUANTIZED:
        raise TypeError(f"dtype must be one of {', '.join(map(str, _QUANTIZED))}, got {dtype}")
    if x.dtype == torch.float64:
        raise TypeError("rms_norm_quantized takes float32, float16 and bfloat16 inputs, got "
                        "torch.float64")
    dim = x.shape[-1]
    group = dim if group_size is None else int(group_size)
    if group < 1 or dim % group:
        raise ValueError(f"group_size must divide {dim}, got {group_size}")
    if _lib.needs_grad(x, weight, residual) or _lib.has_tangent(x, weight, residual):
        raise RuntimeError("rms_norm_quantized has no gradient: use rms_norm, or torch.no_grad()")
    dev = x.device
    q = torch.empty_like(x, dtype=dtype)
    scales = x.new_empty((*x.shape[:-1], dim // group), dtype=torch.float32)
    total = None if residual is None else torch.empty_like(residual)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_rms_norm_quantized(
            *codes, _QUANTIZED[dtype], x.numel() // dim, dim, group, x.data_ptr(),
            _ptr(residual), _ptr(weight), float(eps), q.data_ptr(), scales.data_ptr(),
            _ptr(total), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_rms_norm_quantized")
    return (q, scales) if total is None else (q, scales, total)


class RMSNorm(nn.Module):
    """:func:`rms_norm` with a learned ``weight`` (ones) of ``(dim,)``."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, residual, self.eps)

    def quantized(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                  group_size: Optional[int] = None, dtype: torch.dtype = torch.float8_e4m3fn):
        """:func:`rms_norm_quantized` with this norm's weight."""
        return rms_norm_quantized(x, self.weight, residual, self.eps, group_size, dtype)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, eps={self.eps}"
