"""Short causal convolution over tokens, on sm_100a kernels (``fdwt_causal_conv1d_*`` in
``include/fdwt_b200.h``): every channel has its own few taps.

    p_t = bias + sum_j weight[:, j] x_{t - W + 1 + j},      y = p  or  y = p sigmoid(p)

* :func:`causal_conv1d` -- whole sequences (training, prompts): outputs and the last inputs (the
  state that single tokens carry on), with gradients.
* :func:`causal_conv1d_step` -- one token for each sequence, states updated in place.

It stands before a recurrence such as :func:`~pytorch_morlet_fdwt_b200.selective_scan`, to which
it gives a few neighbouring tokens.  The reference's mixers are not causal and have no counterpart.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .linear_attention import _indexes, _ptr, _rows

__all__ = ["causal_conv1d", "causal_conv1d_step"]

_MAX_WIDTH = 8


class _ConvDesc(ctypes.Structure):
    """ctypes mirror of ``fdwt_conv1d_desc`` (include/fdwt_b200.h)."""

    _fields_ = [("dtype", ctypes.c_int32), ("param_dtype", ctypes.c_int32),
                ("width", ctypes.c_int32), ("silu", ctypes.c_int32), ("batch", ctypes.c_int64),
                ("length", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("x_stride", ctypes.c_int64 * 2), ("dy_stride", ctypes.c_int64 * 2)]


@lru_cache(maxsize=2048)
def _describe(dtype, shape, stride, dy_stride, w_dtype, w_shape, bias, activation, device_index):
    """What a call's types, sizes and strides come to, checked once for each combination on one
    device: the C descriptor, its address and the backward pass's workspace bytes.  ``bias`` is
    the bias's (type, shape) or None."""
    code = _lib.dtype_code(dtype)
    if len(w_shape) != 2 or w_shape[0] != shape[-1]:
        raise ValueError(f"weight must have shape ({shape[-1]}, W), got {tuple(w_shape)}")
    if not 2 <= w_shape[1] <= _MAX_WIDTH:
        raise ValueError(f"weight must have 2 to {_MAX_WIDTH} taps, got {w_shape[1]}")
    if shape[-1] < 1:
        raise ValueError("expected at least one channel")
    if w_dtype != dtype and (w_dtype != torch.float32 or dtype == torch.float64):
        raise TypeError(f"weight must be {dtype} or torch.float32 (torch.float64 for float64 "
                        f"inputs), got {w_dtype}")
    if bias is not None and bias[1] != (shape[-1],):
        raise ValueError(f"bias must have shape ({shape[-1]},), got {tuple(bias[1])}")
    if bias is not None and bias[0] != w_dtype:
        raise TypeError(f"weight and bias must have one type, got {w_dtype} and {bias[0]}")
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    d = _ConvDesc(code, _lib.DTYPES[w_dtype], w_shape[1], activation == "silu", shape[0],
                  shape[1] if len(shape) == 3 else 1, shape[-1])
    d.x_stride[:] = stride[:2] if len(shape) == 3 else (stride[0], 0)
    d.dy_stride[:] = (d.length * d.dim, d.dim) if dy_stride is None else dy_stride[:2]
    at = ctypes.addressof(d)
    with _lib.index_guard(device_index):  # runs of tokens go by the device
        return d, at, int(_lib.load().fdwt_causal_conv1d_backward_workspace(at))


def _plan(x, weight, bias, activation, dy_stride=None):
    return _describe(x.dtype, x.shape, x.stride(), dy_stride, weight.dtype, weight.shape,
                     None if bias is None else (bias.dtype, bias.shape), activation,
                     x.device.index)


def _check_state(state, shape, dtype):
    if tuple(state.shape) != shape or state.dtype != dtype:
        raise ValueError(f"the state must be {dtype} of shape {shape}, got {state.dtype} "
                         f"{tuple(state.shape)}")


def _forward(x, weight, bias, initial, lengths, plan):
    d, desc, _ = plan
    dev = x.device
    y = _lib.empty_like(x)
    final = (x.new_empty((d.batch, d.width - 1, d.dim)) if initial is None
             else _lib.empty_like(initial))
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_causal_conv1d_forward(
            desc, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial), _ptr(lengths),
            y.data_ptr(), final.data_ptr(), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_causal_conv1d_forward")
    return y, final


class _CausalConvFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, lengths, activation, plan):
        ctx.set_materialize_grads(False)
        ctx.activation, ctx.plan = activation, plan
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        return _forward(x, weight, bias, initial, lengths, plan)

    @staticmethod
    @_lib.once
    def backward(ctx, dy, d_final):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        if dy is None and d_final is None:
            return (None,) * 7
        plan = ctx.plan
        d = plan[0]
        dev = x.device
        if dy is None:
            dy = torch.zeros((d.batch, d.length, d.dim), device=dev, dtype=x.dtype)
        elif not dy.is_contiguous():
            dy = _rows(dy)
            plan = _plan(x, weight, bias, ctx.activation, dy.stride())
        if d_final is not None:
            d_final = d_final.contiguous()
        need_x, need_w, need_b, need_i = ctx.needs_input_grad[:4]
        dx = _lib.empty_like(x) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        di = torch.empty_like(initial) if need_i else None
        _, desc, nws = plan
        with _lib.device_guard(dev):
            ws = _lib.workspace(nws if need_w or need_b else 0, dev)
            st = _lib.load().fdwt_causal_conv1d_backward(
                desc, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial), _ptr(lengths),
                dy.data_ptr(), _ptr(d_final), _ptr(dx), _ptr(dw), _ptr(db), _ptr(di), _ptr(ws),
                nws if ws is not None else 0, _lib.raw_stream(dev.index))
        if st:
            _lib.check(st, "fdwt_causal_conv1d_backward")
        return dx, dw, db, di, None, None, None


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  activation: Optional[str] = None, initial_state: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal convolution over whole sequences, each channel with its own taps.

    Args:
        x: ``(B, L, D)``, any strides (a last axis that is not contiguous is copied).
        weight: ``(D, W)``, 2 to 8 taps, the last one that of the token itself; bias: ``(D,)``;
            both of x's type or fp32.
        activation: None or ``"silu"``.
        initial_state: ``(B, W - 1, D)`` of x's type, the inputs before the first token (zeros by
            default).
        lengths: ``(B,)`` int32 or int64, the tokens of each sequence that count (all by default;
            clamped to 0..L).  Outputs after them are zero and the state stops there; the padding
            may hold anything.

    Returns ``(y (B, L, D), final_state (B, W - 1, D))``, differentiable once in x, weight, bias
    and initial_state.  Sums are 32 bits (64 for fp64), rounded once; the gradients' sums over
    tokens are added in a fixed order.
    """
    _lib.require_cuda(x, weight, bias, initial_state, lengths)
    if x.dim() != 3:
        raise ValueError(f"expected (B, L, D) input, got shape {tuple(x.shape)}")
    x, weight = _rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    plan = _plan(x, weight, bias, activation)
    d = plan[0]
    if initial_state is not None:
        _check_state(initial_state, (d.batch, d.width - 1, d.dim), x.dtype)
        initial_state = initial_state.contiguous()
    if lengths is not None:
        lengths = _indexes(lengths, d.batch, 0, d.length, "lengths")
    inputs = (x, weight, bias, initial_state)
    if _lib.needs_grad(*inputs) or _lib.has_tangent(*inputs):
        return _CausalConvFunction.apply(x, weight, bias, initial_state, lengths, activation, plan)
    return _forward(x, weight, bias, initial_state, lengths, plan)


def causal_conv1d_step(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor,
                       bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                       slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`causal_conv1d` for each of B sequences: ``x (B, D)`` -> ``y (B, D)``.

    ``state (N, W - 1, D)``, contiguous and of x's type, is updated in place; ``slots`` names the
    sequences' states as in :func:`~pytorch_morlet_fdwt_b200.linear_attention_step`: without it
    sequence b has state b and N is B, a slot outside ``0..N-1`` touches no state and gives a zero
    output row, and two sequences must not name the same slot.  No gradient: training runs on
    :func:`causal_conv1d`.
    """
    _lib.require_cuda(x, weight, bias, state, slots)
    if x.dim() != 2:
        raise ValueError(f"expected (B, D) input, got shape {tuple(x.shape)}")
    x, weight = _rows(x), weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    d, desc, _ = _plan(x, weight, bias, activation)
    pool = state.shape[0] if state.dim() == 3 and slots is not None else d.batch
    _check_state(state, (pool, d.width - 1, d.dim), x.dtype)
    if not state.is_contiguous():
        raise ValueError("the state is updated in place and must be contiguous")
    if _lib.needs_grad(x, weight, bias, state) or _lib.has_tangent(x, weight, bias, state):
        raise RuntimeError("causal_conv1d_step has no gradient: use causal_conv1d, or "
                           "torch.no_grad()")
    if slots is not None:
        slots = _indexes(slots, d.batch, -1, pool, "slots")
    dev = x.device
    y = _lib.empty_like(x)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_causal_conv1d_step(
            desc, x.data_ptr(), weight.data_ptr(), _ptr(bias), state.data_ptr(), pool,
            _ptr(slots), y.data_ptr(), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_causal_conv1d_step")
    if not state.is_inference():  # written through its pointer: tell autograd
        increment_version(state)
    return y
