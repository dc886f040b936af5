"""Selective state space scan, on sm_100a kernels (``fdwt_selscan_*`` in ``include/fdwt_b200.h``):
a causal token mixer, linear in the sequence length, whose memory goes by the tokens themselves.

    delta_t = dt_t + dt_bias,  or log(1 + exp(dt_t + dt_bias)) with dt_softplus
    h_t = exp(delta_t a) h_{t-1} + delta_t x_t b_t          (N) for each sequence and channel
    y_t = <c_t, h_t> + skip x_t,   times gate_t sigmoid(gate_t) with a gate

* :func:`selective_scan` -- whole sequences (training, prompts): outputs and last states, with
  gradients of every input.
* :func:`selective_scan_step` -- one token for each sequence, states updated in place.

Next to :func:`~pytorch_morlet_fdwt_b200.linear_attention`, whose heads forget at a fixed rate, a
step ``delta_t`` of its own lets each token say how much a channel forgets and takes in.  States,
``a``, ``skip`` and ``dt_bias`` are fp32 (fp64 for fp64 inputs).  The reference's mixers are not
causal and have no counterpart.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .linear_attention import _check_state, _indexes, _ptr, _rows

__all__ = ["selective_scan", "selective_scan_step"]

_MAX_STATES = 128


class _ScanDesc(ctypes.Structure):
    """ctypes mirror of ``fdwt_scan_desc`` (include/fdwt_b200.h)."""

    _fields_ = [("dtype", ctypes.c_int32), ("groups", ctypes.c_int32), ("states", ctypes.c_int32),
                ("dt_softplus", ctypes.c_int32), ("batch", ctypes.c_int64),
                ("length", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("x_stride", ctypes.c_int64 * 2), ("dt_stride", ctypes.c_int64 * 2),
                ("gate_stride", ctypes.c_int64 * 2), ("dy_stride", ctypes.c_int64 * 2),
                ("b_stride", ctypes.c_int64 * 3), ("c_stride", ctypes.c_int64 * 3)]


@lru_cache(maxsize=2048)
def _describe(lead, dtypes, shapes, strides, a_shape, dy_stride, softplus, device_index):
    """What a call's types, sizes and strides come to, checked once for each combination on one
    device: the C descriptor, its address, the bytes of the workspaces and of the kept states, the type
    of states, and the bytes of a backward pass without dL/db and dL/dc; None where a last axis is not contiguous.  In order x, dt, b, c and the gate
    (None without); ``lead`` names the axes before the channels."""
    code = _lib.dtype_code(dtypes[0])
    names = ("x", "dt", "b", "c", "gate")
    for name, dtype in zip(names, dtypes):
        if dtype is not None and dtype != dtypes[0]:
            raise TypeError(f"x, dt, b, c and gate must have one type, got {dtypes[0]} and {dtype} "
                            f"for {name}")
    x, dt, b, c, gate = shapes
    n = len(lead)
    axes = ", ".join(lead)
    if len(x) != n + 1:
        raise ValueError(f"expected x of shape ({axes}, D), got {tuple(x)}")
    for name, s in (("dt", dt), ("gate", gate)):
        if s is not None and s != x:
            raise ValueError(f"{name} must have x's shape {tuple(x)}, got {tuple(s)}")
    if len(b) != n + 2 or b != c or b[:n] != x[:n]:
        raise ValueError(f"b and c must have shape ({axes}, G, N), got {tuple(b)} and {tuple(c)}")
    dim, groups, states = x[-1], b[-2], b[-1]
    if dim < 1 or groups < 1 or dim % groups:
        raise ValueError(f"the channels must be a multiple of the groups, got {dim} and {groups}")
    if not 1 <= states <= _MAX_STATES:
        raise ValueError(f"a channel must have 1 to {_MAX_STATES} states, got {states}")
    if tuple(a_shape) != (dim, states):
        raise ValueError(f"a must have shape ({dim}, {states}), got {tuple(a_shape)}")
    if any(t is not None and t[-1] != 1 and s[-1] != 1 for t, s in zip(strides, shapes)):
        return None
    length = x[1] if n == 2 else 1
    d = _ScanDesc(code, groups, states, bool(softplus), x[0], length, dim)

    def two(stride):  # batch, token; the single-token form has no token axis
        return (0, 0) if stride is None else (stride[:2] if n == 2 else (stride[0], 0))

    def three(stride):
        return stride[:3] if n == 2 else (stride[0], 0, stride[1])

    d.x_stride[:], d.dt_stride[:], d.gate_stride[:] = (two(strides[i]) for i in (0, 1, 4))
    d.b_stride[:], d.c_stride[:] = three(strides[2]), three(strides[3])
    d.dy_stride[:] = (length * dim, dim) if dy_stride is None else dy_stride[:2]
    lib = _lib.load()
    at = ctypes.addressof(d)
    with _lib.index_guard(device_index):  # the cut goes by the device
        return (d, at, int(lib.fdwt_selscan_forward_workspace(at)),
                int(lib.fdwt_selscan_checkpoint_bytes(at)),
                int(lib.fdwt_selscan_backward_workspace(at)),
                torch.float64 if code == 1 else torch.float32,
                int(lib.fdwt_selscan_backward_workspace_least(at)))


def _plan(lead, x, dt, a, b, c, gate, softplus, dy_stride=None):
    dtypes, shapes = (x.dtype, dt.dtype, b.dtype, c.dtype), (x.shape, dt.shape, b.shape, c.shape)
    strides = (x.stride(), dt.stride(), b.stride(), c.stride())
    last = (None, None, None) if gate is None else (gate.dtype, gate.shape, gate.stride())
    return _describe(lead, (*dtypes, last[0]), (*shapes, last[1]), (*strides, last[2]), a.shape,
                     dy_stride, bool(softplus), x.get_device())


_SEQUENCE, _TOKEN = ("B", "L"), ("B",)


def _parameter(name: str, t: Optional[torch.Tensor], shape, dtype) -> Optional[torch.Tensor]:
    """``t`` contiguous and in the states' type (a cast that autograd follows)."""
    if t is None or (t.dtype is dtype and t.shape == shape and t.is_contiguous()):
        return t
    if tuple(t.shape) != shape or not t.is_floating_point():
        raise ValueError(f"{name} must be floating point of shape {shape}, got {t.dtype} "
                         f"{tuple(t.shape)}")
    return t.to(dtype).contiguous()


def _forward(x, dt, a, b, c, skip, gate, dt_bias, initial, lengths, plan, keep: bool):
    d, desc, nws, ncheck, _, acc, _ = plan
    dev = x.device
    y = _lib.empty_like(x)
    final = (x.new_empty((d.batch, d.dim, d.states), dtype=acc) if initial is None
             else _lib.empty_like(initial))
    check = x.new_empty(ncheck, dtype=torch.uint8) if keep else None
    with _lib.device_guard(dev):
        ws = _lib.workspace(nws, dev)
        st = _lib.load().fdwt_selscan_forward(
            desc, x.data_ptr(), dt.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(),
            _ptr(skip), _ptr(gate), _ptr(dt_bias), _ptr(initial), _ptr(lengths), y.data_ptr(),
            final.data_ptr(), _ptr(check), _ptr(ws), nws, _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_selscan_forward")
    return y, final, check


class _SelectiveScanFunction(torch.autograd.Function):
    """The forward pass keeps the states before every eighth token (4 N bytes an eighth token and
    channel), from which the backward pass forms the others again."""

    @staticmethod
    def forward(ctx, x, dt, a, b, c, skip, gate, dt_bias, initial, lengths, softplus, plan):
        ctx.set_materialize_grads(False)
        ctx.softplus, ctx.plan = softplus, plan
        y, final, check = _forward(x, dt, a, b, c, skip, gate, dt_bias, initial, lengths, plan,
                                   True)
        ctx.save_for_backward(x, dt, a, b, c, skip, gate, dt_bias, initial, lengths, check)
        return y, final

    @staticmethod
    @_lib.once
    def backward(ctx, dy, d_final):
        x, dt, a, b, c, skip, gate, dt_bias, initial, lengths, check = ctx.saved_tensors
        if dy is None and d_final is None:
            return (None,) * 12
        plan = ctx.plan
        d, dev = plan[0], x.device
        if dy is None:
            dy = torch.zeros((d.batch, d.length, d.dim), device=dev, dtype=x.dtype)
        elif not dy.is_contiguous():
            dy = _rows(dy)
            plan = _plan(_SEQUENCE, x, dt, a, b, c, gate, ctx.softplus, dy.stride())
        if d_final is not None:
            d_final = d_final.contiguous()
        _, _, need_a, need_b, need_c, need_skip, _, need_bias, need_i = ctx.needs_input_grad[:9]
        like = _lib.empty_like
        dx, ddt, dgate = like(x), like(dt), None if gate is None else like(gate)
        da = like(a) if need_a else None
        db = like(b) if need_b else None
        dc = like(c) if need_c else None
        dskip = like(skip) if need_skip else None
        dbias = like(dt_bias) if need_bias else None
        di = like(initial) if need_i else None
        _, desc, _, _, nws, _, least = plan
        if not (need_b or need_c):
            nws = least
        with _lib.device_guard(dev):
            ws = _lib.workspace(nws, dev)
            st = _lib.load().fdwt_selscan_backward(
                desc, x.data_ptr(), dt.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(),
                _ptr(skip), _ptr(gate), _ptr(dt_bias), _ptr(lengths), check.data_ptr(),
                dy.data_ptr(), _ptr(d_final), dx.data_ptr(), ddt.data_ptr(), _ptr(da), _ptr(db),
                _ptr(dc), _ptr(dskip), _ptr(dgate), _ptr(dbias), _ptr(di), _ptr(ws), nws,
                _lib.raw_stream(dev.index))
        if st:
            _lib.check(st, "fdwt_selscan_backward")
        return dx, ddt, da, db, dc, dskip, dgate, dbias, di, None, None, None


def selective_scan(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                   c: torch.Tensor, skip: Optional[torch.Tensor] = None,
                   gate: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   dt_softplus: bool = False, initial_state: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Selective scan over whole sequences.

    Args:
        x, dt: ``(B, L, D)``, inputs and steps; b, c: ``(B, L, G, N)``, shared by the channels of a
            group (channel d reads group ``d // (D // G)``); gate: ``(B, L, D)``; one type, any
            strides (a last axis that is not contiguous is copied).  Up to 128 states N.
        a: ``(D, N)``, the rates (negative: the state decays; finite or ``-inf``); skip, dt_bias:
            ``(D,)``; taken in fp32 (fp64 for fp64 inputs).
        dt_softplus: the step is ``log(1 + exp(dt + dt_bias))`` in place of ``dt + dt_bias``; a dt
            of ``-inf`` is then a step of zero, which keeps the state.
        initial_state: ``(B, D, N)`` fp32 (fp64 for fp64 inputs), zeros by default.
        lengths: ``(B,)`` int32 or int64, the tokens of each sequence that count (all by default;
            clamped to 0..L).  Outputs after them are zero and the state stops there; the padding
            may hold anything.

    Returns ``(y (B, L, D), final_state (B, D, N))``, differentiable once in every input but the
    lengths.  fp16 and bf16 inputs are computed in 32 bits, states too, and the result rounded
    once.  An infinity or NaN reaches the outputs of its token and later ones only (an infinity may
    reach them as a NaN).  A call whose inputs need gradients keeps ``L / 8`` states of every channel
    for the backward pass, which has up to 1 GiB of scratch besides (or one tile's, if that is more).
    """
    _lib.require_cuda(x, dt, a, b, c, skip, gate, dt_bias, initial_state, lengths)
    plan = _plan(_SEQUENCE, x, dt, a, b, c, gate, dt_softplus)
    if plan is None:
        x, dt, b, c = _rows(x), _rows(dt), _rows(b), _rows(c)
        gate = None if gate is None else _rows(gate)
        plan = _plan(_SEQUENCE, x, dt, a, b, c, gate, dt_softplus)
    d, acc = plan[0], plan[5]
    a = _parameter("a", a, (d.dim, d.states), acc)
    skip = _parameter("skip", skip, (d.dim,), acc)
    dt_bias = _parameter("dt_bias", dt_bias, (d.dim,), acc)
    if initial_state is not None:
        _check_state(initial_state, (d.batch, d.dim, d.states), acc)
        initial_state = initial_state.contiguous()
    if lengths is not None:
        lengths = _indexes(lengths, d.batch, 0, d.length, "lengths")
    inputs = (x, dt, a, b, c, skip, gate, dt_bias, initial_state)
    if _lib.needs_grad(*inputs) or _lib.has_tangent(*inputs):
        return _SelectiveScanFunction.apply(*inputs, lengths, bool(dt_softplus), plan)
    return _forward(*inputs, lengths, plan, False)[:2]


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                        c: torch.Tensor, state: torch.Tensor,
                        skip: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                        slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`selective_scan` for each of B sequences: ``x, dt, gate (B, D)``,
    ``b, c (B, G, N)`` -> ``y (B, D)``.

    ``state (S, D, N)``, contiguous fp32 (fp64 for fp64 inputs), is updated in place; ``slots``
    names the sequences' states as in :func:`~pytorch_morlet_fdwt_b200.linear_attention_step`:
    without it sequence b has state b and S is B, a slot outside ``0..S-1`` touches no state and
    gives a zero output row, and two sequences must not name the same slot.  No gradient: training
    runs on :func:`selective_scan`.
    """
    _lib.require_cuda(x, dt, a, b, c, state, skip, gate, dt_bias, slots)
    plan = _plan(_TOKEN, x, dt, a, b, c, gate, dt_softplus)
    if plan is None:
        x, dt, b, c = _rows(x), _rows(dt), _rows(b), _rows(c)
        gate = None if gate is None else _rows(gate)
        plan = _plan(_TOKEN, x, dt, a, b, c, gate, dt_softplus)
    d, desc, _, _, _, acc, _ = plan
    a = _parameter("a", a, (d.dim, d.states), acc)
    skip = _parameter("skip", skip, (d.dim,), acc)
    dt_bias = _parameter("dt_bias", dt_bias, (d.dim,), acc)
    pool = state.shape[0] if state.dim() == 3 and slots is not None else d.batch
    _check_state(state, (pool, d.dim, d.states), acc)
    if not state.is_contiguous():
        raise ValueError("the state is updated in place and must be contiguous")
    inputs = (x, dt, a, b, c, skip, gate, dt_bias, state)
    if _lib.needs_grad(*inputs) or _lib.has_tangent(*inputs):
        raise RuntimeError("selective_scan_step has no gradient: use selective_scan, or "
                           "torch.no_grad()")
    if slots is not None:
        slots = _indexes(slots, d.batch, -1, pool, "slots")
    dev = x.device
    y = _lib.empty_like(x)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_selscan_step(
            desc, x.data_ptr(), dt.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(),
            _ptr(skip), _ptr(gate), _ptr(dt_bias), state.data_ptr(), pool, _ptr(slots),
            y.data_ptr(), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_selscan_step")
    if not state.is_inference():  # written through its pointer: tell autograd
        increment_version(state)
    return y
