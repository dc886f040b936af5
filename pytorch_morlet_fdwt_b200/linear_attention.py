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


@lru_cache(maxsize=1024)
def _describe(dtype, batch, length, heads, kv_heads, dk, dv, qs, ks, vs, os, scale,
              device_index) -> Tuple[_Desc, int, int, int]:
    """The C descriptor of a call, its address and the workspace bytes of the forward and the
    backward pass: pure functions of the sizes on one device (the library only reads it)."""
    d = _Desc(dtype, heads, kv_heads, dk, dv, batch, length)
    d.q_stride[:], d.k_stride[:], d.v_stride[:], d.o_stride[:] = qs, ks, vs, os
    d.scale = scale
    lib = _lib.load()
    at = ctypes.addressof(d)
    return (d, at, int(lib.fdwt_linattn_forward_workspace(at)),
            int(lib.fdwt_linattn_backward_workspace(at)))


def _acc(dtype: torch.dtype) -> torch.dtype:
    return torch.float64 if dtype == torch.float64 else torch.float32


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous last axis (any other strides are taken as they are)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(t: torch.Tensor) -> Tuple[int, int, int]:
    return t.stride()[:3]


def _check_heads(q, k, v, log_decay, names):
    """Types and sizes shared by both forms; the head axis is the last but one."""
    _lib.require_cuda(q, k, v, log_decay)
    code = _lib.dtype_code(q.dtype)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != len(names) or len(ks) != len(qs) or len(vs) != len(qs):
        raise ValueError(f"expected q, k, v of shape ({', '.join(names)}), got {tuple(qs)}, "
                         f"{tuple(ks)}, {tuple(vs)}")
    if ks[:-2] != qs[:-2] or vs[:-1] != ks[:-1]:
        raise ValueError(f"q, k and v must agree in {', '.join(names[:-2])} and k and v in their "
                         f"heads, got {tuple(qs)}, {tuple(ks)}, {tuple(vs)}")
    heads, dk = qs[-2:]
    kv_heads, dv = vs[-2:]
    if ks[-1] != dk:
        raise ValueError(f"q and k must have one head size, got {dk} and {ks[-1]}")
    if not (1 <= dk <= _MAX_HEAD and 1 <= dv <= _MAX_HEAD):
        raise ValueError(f"head sizes must be 1 to {_MAX_HEAD}, got {dk} and {dv}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"the query heads must be a multiple of the key and value heads, got "
                         f"{heads} and {kv_heads}")
    if log_decay.shape != (heads,) or not log_decay.is_floating_point():
        raise ValueError(f"log_decay must be floating point of shape ({heads},), got "
                         f"{log_decay.dtype} {tuple(log_decay.shape)}")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a fixed schedule without a gradient; detach it")
    return code, heads, kv_heads, dk, dv


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


def _forward(q, k, v, log_decay, initial, lengths, scale, sizes):
    code, heads, kv_heads, dk, dv = sizes
    batch, length = q.shape[:2]
    dev = q.device
    out = torch.empty((batch, length, heads, dv), device=dev, dtype=q.dtype)
    final = torch.empty((batch, heads, dk, dv), device=dev, dtype=log_decay.dtype)
    with _lib.device_guard(dev):
        _, desc, nws, _ = _describe(code, batch, length, heads, kv_heads, dk, dv, _strides(q),
                                    _strides(k), _strides(v), _strides(out), scale, dev.index)
        ws = _lib.workspace(nws, dev)
        st = _lib.load().fdwt_linattn_forward(
            desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
            None if initial is None else initial.data_ptr(),
            None if lengths is None else lengths.data_ptr(), out.data_ptr(), final.data_ptr(),
            None if ws is None else ws.data_ptr(), nws, _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_linattn_forward")
    if config.check_device_errors:
        _lib.check_device_error("fdwt_linattn_forward")
    return out, final


class _LinearAttentionFunction(torch.autograd.Function):
    """The backward pass is the same operator three times, with other operands and, for k and v,
    back in time (one C call)."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, scale, sizes):
        ctx.set_materialize_grads(False)
        ctx.scale, ctx.sizes = scale, sizes
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths)
        return _forward(q, k, v, log_decay, initial, lengths, scale, sizes)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, log_decay, initial, lengths = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 8
        code, heads, kv_heads, dk, dv = ctx.sizes
        batch, length = q.shape[:2]
        dev = q.device
        if d_out is None:
            d_out = torch.zeros((batch, length, heads, dv), device=dev, dtype=q.dtype)
        d_out = _rows(d_out)
        d_final = None if d_final is None else d_final.contiguous()
        dq, dkk, dvv = (torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, k, v))
        need_state = ctx.needs_input_grad[4]
        d_initial = torch.empty_like(initial) if need_state else None
        with _lib.device_guard(dev):
            _, desc, _, nws = _describe(code, batch, length, heads, kv_heads, dk, dv, _strides(q),
                                        _strides(k), _strides(v), _strides(d_out), ctx.scale,
                                        dev.index)
            ws = _lib.workspace(nws, dev)
            st = _lib.load().fdwt_linattn_backward(
                desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                None if initial is None else initial.data_ptr(),
                None if lengths is None else lengths.data_ptr(), d_out.data_ptr(),
                None if d_final is None else d_final.data_ptr(), dq.data_ptr(), dkk.data_ptr(),
                dvv.data_ptr(), None if d_initial is None else d_initial.data_ptr(),
                None if ws is None else ws.data_ptr(), nws, _lib.raw_stream(dev.index))
        if st:
            _lib.check(st, "fdwt_linattn_backward")
        if config.check_device_errors:
            _lib.check_device_error("fdwt_linattn_backward")
        return dq, dkk, dvv, None, d_initial, None, None, None


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
    and initial_state.  fp16 and bf16 round the scores and the state's copy that multiplies q to
    16 bits; the state itself is fp32.
    """
    sizes = _check_heads(q, k, v, log_decay, ("B", "L", "H", "D"))
    code, heads, kv_heads, dk, dv = sizes
    batch, length = q.shape[:2]
    acc = _acc(q.dtype)
    if log_decay.dtype != acc or not log_decay.is_contiguous():
        log_decay = log_decay.to(acc).contiguous()
    if initial_state is not None:
        _lib.require_cuda(q, initial_state)
        _check_state(initial_state, (batch, heads, dk, dv), acc)
        initial_state = initial_state.contiguous()
    if lengths is not None:
        _lib.require_cuda(q, lengths)
        lengths = _indexes(lengths, batch, 0, length, "lengths")
    scale = float(dk) ** -0.5 if scale is None else float(scale)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (
            initial_state is not None and initial_state.requires_grad)):
        return _LinearAttentionFunction.apply(q, k, v, log_decay, initial_state, lengths, scale,
                                              sizes)
    return _forward(q, k, v, log_decay, initial_state, lengths, scale, sizes)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          log_decay: torch.Tensor, state: torch.Tensor,
                          scale: Optional[float] = None,
                          slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of :func:`linear_attention` for each of B sequences: ``q (B, H, Dk)``,
    ``k (B, Hkv, Dk)``, ``v (B, Hkv, Dv)`` -> ``out (B, H, Dv)``.

    ``state (N, H, Dk, Dv)``, contiguous fp32 (fp64 for fp64 inputs), is updated in place.
    Without ``slots`` sequence b has state b and N is B.  ``slots (B,)``, int32 or int64, names
    each sequence's state in a pool; a slot outside ``0..N-1`` (-1 for an empty row of a batch)
    touches no state and gives a zero output row.  Two sequences must not name the same slot.
    No gradient: training runs on :func:`linear_attention`.
    """
    sizes = _check_heads(q, k, v, log_decay, ("B", "H", "D"))
    code, heads, kv_heads, dk, dv = sizes
    batch = q.shape[0]
    acc = _acc(q.dtype)
    _lib.require_cuda(q, state, slots)
    pool = state.shape[0] if state.dim() == 4 and slots is not None else batch
    _check_state(state, (pool, heads, dk, dv), acc)
    if not state.is_contiguous():
        raise ValueError("the state is updated in place and must be contiguous")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or state.requires_grad):
        raise RuntimeError("linear_attention_step has no gradient: use linear_attention, or "
                           "torch.no_grad()")
    if slots is not None:
        slots = _indexes(slots, batch, -1, pool, "slots")
    if log_decay.dtype != acc or not log_decay.is_contiguous():
        log_decay = log_decay.to(acc).contiguous()
    scale = float(dk) ** -0.5 if scale is None else float(scale)
    q, k, v = _rows(q), _rows(k), _rows(v)
    dev = q.device
    out = torch.empty((batch, heads, dv), device=dev, dtype=q.dtype)
    # (batch, head) strides with an unused token stride between them
    with _lib.device_guard(dev):
        _, desc, _, _ = _describe(code, batch, 1, heads, kv_heads, dk, dv,
                                  (q.stride(0), 0, q.stride(1)), (k.stride(0), 0, k.stride(1)),
                                  (v.stride(0), 0, v.stride(1)), (heads * dv, 0, dv), scale,
                                  dev.index)
        st = _lib.load().fdwt_linattn_step(
            desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
            state.data_ptr(), pool, None if slots is None else slots.data_ptr(), out.data_ptr(),
            _lib.raw_stream(dev.index))
    if st:
        _lib.check(st, "fdwt_linattn_step")
    return out
