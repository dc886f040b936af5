"""Linear attention with a decay for each head, on sm_100a kernels (``fdwt_linattn_*`` in
``include/fdwt_b200.h``): a causal token mixer, linear in the sequence length, whose state takes
the place of a key-value cache.

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T        (Dk, Dv) for each sequence and head
    o_t = scale * q_t^T S_t

* :func:`linear_attention` -- whole sequences (training, prompts): outputs and last states, with
  gradients of q, k, v and the initial states.
* :func:`linear_attention_step` -- one token for each sequence, states updated in place.

``log_decay`` is a fixed schedule of the heads (zero or negative; ``-inf`` forgets everything),
not a parameter: it has no gradient.  States are fp32 (fp64 for fp64 inputs).  The reference's
mixers are not causal and have no counterpart of this.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib, config

__all__ = ["linear_attention", "linear_attention_step"]

_MAX_HEAD = 256


class _Desc(ctypes.Structure):
    """ctypes mirror of ``fdwt_linattn_desc`` (include/fdwt_b200.h)."""

    _fields_ = [("dtype", ctypes.c_int32), ("heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("dk", ctypes.c_int32), ("dv", ctypes.c_int32), ("batch", ctypes.c_int64),
                ("length", ctypes.c_int64), ("q_stride", ctypes.c_int64 * 3),
                ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
                ("o_stride", ctypes.c_int64 * 3), ("scale", ctypes.c_double)]


@lru_cache(maxsize=2048)
def _describe(names, dtypes, shapes, strides, out_stride, scale, device_index):
    """What a call's types, sizes and strides come to, checked once for each combination on one
    device: the C descriptor and its address, the workspace bytes of the forward and the backward
    pass, and the type of states.  The shapes and strides are (..., heads, size) of q, k and v;
    ``out_stride`` None stands for a contiguous result."""
    code = _lib.dtype_code(dtypes[0])
    if dtypes[1] != dtypes[0] or dtypes[2] != dtypes[0]:
        raise TypeError("q, k and v must have one type, got "
                        f"{dtypes[0]}, {dtypes[1]}, {dtypes[2]}")
    qs, ks, vs = (tuple(s) for s in shapes)
    if not len(qs) == len(ks) == len(vs) == len(names):
        raise ValueError(f"expected q, k, v of shape ({', '.join(names)}), got {qs}, {ks}, {vs}")
    if ks[:-2] != qs[:-2] or vs[:-1] != ks[:-1]:
        raise ValueError(f"q, k and v must agree in {', '.join(names[:-2])} and k and v in their "
                         f"heads, got {qs}, {ks}, {vs}")
    heads, dk = qs[-2:]
    kv_heads, dv = vs[-2:]
    if ks[-1] != dk:
        raise ValueError(f"q and k must have one head size, got {dk} and {ks[-1]}")
    if not (1 <= dk <= _MAX_HEAD and 1 <= dv <= _MAX_HEAD):
        raise ValueError(f"head sizes must be 1 to {_MAX_HEAD}, got {dk} and {dv}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"the query heads must be a multiple of the key and value heads, got "
                         f"{heads} and {kv_heads}")
    batch, length = qs[0], qs[1] if len(qs) == 4 else 1

    def three(stride):  # batch, token, head; the single-token form has no token axis
        return stride[:3] if len(qs) == 4 else (stride[0], 0, stride[1])

    d = _Desc(code, heads, kv_heads, dk, dv, batch, length)
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = (three(s) for s in strides)
    d.o_stride[:] = ((length * heads * dv, heads * dv, dv) if out_stride is None
                     else three(out_stride))
    d.scale = float(dk) ** -0.5 if scale is None else float(scale)
    lib = _lib.load()
    at = ctypes.addressof(d)
    state = torch.float64 if code == 1 else torch.float32
    return (d, at, int(lib.fdwt_linattn_forward_workspace(at)),
            int(lib.fdwt_linattn_backward_workspace(at)), state)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous last axis (any other strides are taken as they are)."""
    return t if t.dim() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _plan(names, q, k, v, scale, out_stride=None):
    if scale is not None and type(scale) is not float:
        # a number by value: a tensor would be looked up by its identity
        if isinstance(scale, torch.Tensor) and scale.requires_grad:
            raise ValueError("scale is a number without a gradient; detach it")
        scale = float(scale)
    return _describe(names, (q.dtype, k.dtype, v.dtype), (q.shape, k.shape, v.shape),
                     (q.stride(), k.stride(), v.stride()), out_stride, scale, q.device.index)


def _schedule(log_decay, heads: int, dtype: torch.dtype) -> torch.Tensor:
    """``log_decay (heads,)`` contiguous in the states' type."""
    if log_decay.shape != (heads,) or not log_decay.is_floating_point():
        raise ValueError(f"log_decay must be floating point of shape ({heads},), got "
                         f"{log_decay.dtype} {tuple(log_decay.shape)}")
    if log_decay.requires_grad or _lib.has_tangent(log_decay):
        raise ValueError("log_decay is a fixed schedule without a gradient; detach it")
    if log_decay.dtype != dtype or not log_decay.is_contiguous():
        log_decay = log_decay.to(dtype).contiguous()
    return log_decay


def _check_state(state, shape, dtype):
    if tuple(state.shape) != shape or state.dtype != dtype:
        raise ValueError(f"the state must be {dtype} of shape {shape}, got {state.dtype} "
                         f"{tuple(state.shape)}")


def _indexes(t: torch.Tensor, count: int, low: int, high: int, name: str) -> torch.Tensor:
    """A ``(count,)`` integer tensor as contiguous int32 (wider types clamped to low..high)."""
    if t.shape != (count,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64 of shape ({count},), got {t.dtype} "
                         f"{tuple(t.shape)}")
    if t.dtype == torch.int64:
        t = t.clamp(low, high).to(torch.int32)
    return t.contiguous()


_SEQUENCE, _TOKEN = ("B", "L", "H", "D"), ("B", "H", "D")


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _forward(q, k, v, log_decay, initial, lengths, plan):
    d, desc, nws, _, acc = plan
    dev = q.device
    out = torch.empty((d.batch, d.length, d.heads, d.dv), device=dev, dtype=q.dtype)
    final = torch.empty((d.batch, d.heads, d.dk, d.dv), device=dev, dtype=acc)
    with _lib.device_guard(dev):
        ws = _lib.workspace(nws, dev)
        st = _lib.load().fdwt_linattn_forward(
            desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _ptr(initial),
            _ptr(lengths), out.data_ptr(), final.data_ptr(), _ptr(ws), nws,
            _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_linattn_forward")
    if config.check_device_errors:
        _lib.check_device_error("fdwt_linattn_forward")
    return out, final


class _LinearAttentionFunction(torch.autograd.Function):
    """The backward pass is the same operator three times, with other operands and, for k and v,
    back in time (one C call)."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, plan):
        ctx.set_materialize_grads(False)
        ctx.plan = plan
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths)
        return _forward(q, k, v, log_decay, initial, lengths, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, log_decay, initial, lengths = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 7
        plan = ctx.plan
        d = plan[0]
        dev = q.device
        if d_out is None:
            d_out = torch.zeros((d.batch, d.length, d.heads, d.dv), device=dev, dtype=q.dtype)
        elif not d_out.is_contiguous():
            d_out = _rows(d_out)
            plan = _plan(_SEQUENCE, q, k, v, d.scale, d_out.stride())
        if d_final is not None:
            d_final = d_final.contiguous()
        dq, dkk, dvv = (torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, k, v))
        d_initial = torch.empty_like(initial) if ctx.needs_input_grad[4] else None
        _, desc, _, nws, _ = plan
        with _lib.device_guard(dev):
            ws = _lib.workspace(nws, dev)
            st = _lib.load().fdwt_linattn_backward(
                desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                _ptr(initial), _ptr(lengths), d_out.data_ptr(), _ptr(d_final), dq.data_ptr(),
                dkk.data_ptr(), dvv.data_ptr(), _ptr(d_initial), _ptr(ws), nws,
                _lib.raw_stream(dev.index))
        if st:
            _lib.check(st, "fdwt_linattn_backward")
        if config.check_device_errors:
            _lib.check_device_error("fdwt_linattn_backward")
        return dq, dkk, dvv, None, d_initial, None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     scale: Optional[float] = None,
                     initial_state: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Causal linear attention with a decay for each head over whole sequences.

    Args:
        q: ``(B, L, H, Dk)``; k: ``(B, L, Hkv, Dk)``; v: ``(B, L, Hkv, Dv)``, one type, any
            strides (a last axis that is not contiguous is copied).  ``H`` is a multiple of
            ``Hkv``: query head h reads key and value head ``h // (H // Hkv)``.  Head sizes up
            to 256.
        log_decay: ``(H,)``, the log of each head's decay a token.
        scale: factor of the outputs, ``Dk ** -0.5`` by default.
        initial_state: ``(B, H, Dk, Dv)`` fp32 (fp64 for fp64 inputs), zeros by default.
        lengths: ``(B,)`` int32 or int64, the tokens of each sequence that count (all by default;
            clamped to 0..L).  Outputs after them are zero and the state stops there; the padding
            may hold anything.

    Returns ``(out (B, L, H, Dv), final_state (B, H, Dk, Dv))``, differentiable once in q, k, v
    and initial_state.  fp16 and bf16 inputs are computed to 32 bits, states too, and the result
    rounded once.  An infinity or NaN reaches the outputs of its token and later ones only.

    The kernels for fp16 and bf16 wait on copies with a time limit (about a second; a machine in
    order never gets near it).  Where one runs out the results are incomplete and the call does
    not know: :func:`~pytorch_morlet_fdwt_b200._lib.device_error` does, and with
    ``config.check_device_errors`` every call asks it, synchronising the device, and raises.
    """
    _lib.require_cuda(q, k, v, log_decay, initial_state, lengths)
    q, k, v = _rows(q), _rows(k), _rows(v)
    plan = _plan(_SEQUENCE, q, k, v, scale)
    d, acc = plan[0], plan[4]
    log_decay = _schedule(log_decay, d.heads, acc)
    needs = q.requires_grad or k.requires_grad or v.requires_grad
    if initial_state is not None:
        _check_state(initial_state, (d.batch, d.heads, d.dk, d.dv), acc)
        initial_state = initial_state.contiguous()
        needs = needs or initial_state.requires_grad
    if lengths is not None:
        lengths = _indexes(lengths, d.batch, 0, d.length, "lengths")
    if (needs and torch.is_grad_enabled()) or _lib.has_tangent(q, k, v, initial_state):
        return _LinearAttentionFunction.apply(q, k, v, log_decay, initial_state, lengths, plan)
    return _forward(q, k, v, log_decay, initial_state, lengths, plan)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          log_decay: torch.Tensor, state: torch.Tensor,
                          scale: Optional[float] = None,
                          slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`linear_attention` for each of B sequences: ``q (B, H, Dk)``,
    ``k (B, Hkv, Dk)``, ``v (B, Hkv, Dv)`` -> ``out (B, H, Dv)``.

    ``state (N, H, Dk, Dv)``, contiguous fp32 (fp64 for fp64 inputs), is updated in place (as by
    any in-place operation, a graph that saved it then raises in its backward pass).
    Without ``slots`` sequence b has state b and N is B.  ``slots (B,)``, int32 or int64, names
    each sequence's state in a pool; a slot outside ``0..N-1`` (-1 for an empty row of a batch)
    touches no state and gives a zero output row.  Two sequences must not name the same slot.
    No gradient: training runs on :func:`linear_attention`.
    """
    _lib.require_cuda(q, k, v, log_decay, state, slots)
    q, k, v = _rows(q), _rows(k), _rows(v)
    d, desc, _, _, acc = _plan(_TOKEN, q, k, v, scale)
    log_decay = _schedule(log_decay, d.heads, acc)
    pool = state.shape[0] if state.dim() == 4 and slots is not None else d.batch
    _check_state(state, (pool, d.heads, d.dk, d.dv), acc)
    if not state.is_contiguous():
        raise ValueError("the state is updated in place and must be contiguous")
    if ((q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad)
            and torch.is_grad_enabled()) or _lib.has_tangent(q, k, v, state):
        raise RuntimeError("linear_attention_step has no gradient: use linear_attention, or "
                           "torch.no_grad()")
    if slots is not None:
        slots = _indexes(slots, d.batch, -1, pool, "slots")
    dev = q.device
    out = torch.empty((d.batch, d.heads, d.dv), device=dev, dtype=q.dtype)
    with _lib.device_guard(dev):
        st = _lib.load().fdwt_linattn_step(
            desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
            state.data_ptr(), pool, _ptr(slots), out.data_ptr(), _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_linattn_step")
    # written through its pointer: tell autograd, so that a graph that saved this state raises in
    # its backward pass (inference tensors keep no count and are in no graph)
    if not state.is_inference():
        increment_version(state)
    return out
