"""selective_scan and selective_scan_step at the ends of the step's range: with dt_softplus a dt of
-inf is a step of exactly zero, and one of any size its own step.

log(1 + e^v) is 0 for v = -inf and, rounded, for v = -1e4, and its slope with it, so that a call with
the one gives bit by bit what a call with the other gives.  Large |v| go by the tolerances of the
scan's other tests."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

from .test_selective_scan_gpu import (BF16, DEV, F16, F32, F64, NAMES, _acc, _call, _case, _check,
                                      _reference)

pytestmark = pytest.mark.gpu


def _outcome(s, names):
    for k in names:
        s[k] = s[k].detach().requires_grad_()
    y, final = _call(s)
    torch.manual_seed(3)
    dy, df = torch.randn_like(y), torch.randn_like(final)
    return (y.detach(), final.detach(),
            *torch.autograd.grad((y, final), [s[k] for k in names], (dy, df)))


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("L,D,N,options", [(1, 8, 4, {}), (21, 40, 16, {}), (37, 33, 5, {"bias": False}),
                                           (70, 24, 100, {"gate": False}),
                                           (2100, 32, 16, {"lengths": [2100, 1777]})])
def test_a_step_of_minus_infinity_is_no_step(L, D, N, options, dtype):
    s = _case(2, L, D, N, 1, dtype, seed=L, **options)
    names = [k for k in NAMES if s[k] is not None]
    off = torch.rand(2, L, D, device=DEV) < 0.3
    off[:, ::5] = True  # whole tokens, the first among them
    got = _outcome(s | {"dt": s["dt"].masked_fill(off, float("-inf"))}, names)
    want = _outcome(s | {"dt": s["dt"].masked_fill(off, -1e4)}, names)
    for name, p, q in zip(("y", "final", *names), got, want):
        assert torch.isfinite(p).all(), name
        assert torch.equal(p, q), name
    assert not got[2 + names.index("dt")][off].any()


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("N", [16, 5])
def test_a_single_token_without_a_step_keeps_its_state(N, dtype):
    s = _case(3, 1, 40, N, 1, dtype, seed=N)
    state = s["initial"].clone()
    token = {k: s[k][:, 0] for k in ("x", "dt", "b", "c", "gate")}
    y = F.selective_scan_step(token["x"], torch.full_like(token["dt"], float("-inf")), s["a"],
                              token["b"], token["c"], state, s["skip"], token["gate"], s["dt_bias"],
                              True)
    assert torch.equal(state, s["initial"]) and torch.isfinite(y).all()
    ref = _reference(s | {"dt": torch.full_like(s["dt"], -1e4)})
    _check(y, tuple(t[:, 0] for t in ref["y"]), dtype, "y", _acc(dtype))


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("bias", [False, True])
def test_large_steps_of_both_signs(dtype, bias):
    s = _case(2, 40, 48, 16, 1, dtype, seed=5, bias=bias)
    torch.manual_seed(6)
    size = torch.empty(2, 40, 48, device=DEV).uniform_(20, 200)
    s["dt"] = (size * torch.where(torch.rand_like(size) < 0.5, -1.0, 1.0)).to(dtype)
    s["x"] = s["x"] / 16  # (and dy: fp16 holds up to 65504)
    names = [k for k in NAMES if s[k] is not None]
    for k in names:
        s[k].requires_grad_()
    y, final = _call(s)
    dy, df = torch.randn_like(y) / 16, torch.randn_like(final)
    ref = _reference(s, dy, df)
    _check(y.detach(), ref["y"], dtype, "y", _acc(dtype))
    _check(final.detach(), ref["final"], final.dtype, "final")
    grads = torch.autograd.grad((y, final), [s[k] for k in names], (dy, df))
    for k, g in zip(names, grads):
        _check(g, ref[k], s[k].dtype, f"dL/d{k}", _acc(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_largest_steps_are_finite(dtype):
    """3e38 (rounded to the type) is its own step: with x = b = 1/4 the state is a 16th of it.  The
    state: two products, exact by powers of two."""
    step = torch.tensor(3e38, device=DEV).to(dtype)
    quarter = torch.full((1, 3, 8), 0.25, device=DEV).to(dtype)
    dt = torch.full_like(quarter, float(step))
    bc = torch.full((1, 3, 1, 4), 0.25, device=DEV).to(dtype)
    a = -torch.ones(8, 4, device=DEV)
    y, final = F.selective_scan(quarter, dt, a, bc, bc * 2.0 ** -60, dt_softplus=True)
    assert torch.isfinite(y).all() and torch.equal(final, (step.float() / 16).expand_as(final))
    state = torch.ones(1, 8, 4, device=DEV)
    F.selective_scan_step(quarter[:, 0], dt[:, 0], a, bc[:, 0], bc[:, 0], state, dt_softplus=True)
    assert torch.equal(state, final)
