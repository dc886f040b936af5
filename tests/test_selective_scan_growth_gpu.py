"""selective_scan with rates above zero (or steps below) over sequences long enough to be cut: a state of
zero stays zero however much the segments after it would grow one, so that a call over a long stretch of
zeros gives what the call without the stretch gives, bit by bit."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, F32, F16, BF16 = torch.float64, torch.float32, torch.float16, torch.bfloat16
L, D, N, TAIL = 8192, 64, 16, 64


def _inputs(dtype, down):
    """Steps of 1 (or, with rates below zero, -1) and rates that double a state every 1 to 3 tokens."""
    torch.manual_seed(2)
    wide = F64 if dtype == F64 else F32
    x, b, c = (torch.randn(1, L, *s, device=DEV).to(dtype) for s in ((D,), (1, N), (1, N)))
    dt = torch.full((1, L, D), -1.0 if down else 1.0, device=DEV, dtype=dtype)
    a = (0.25 + 0.5 * torch.rand(D, N, device=DEV)).to(wide) * (-1 if down else 1)
    return x, dt, a, b, c


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("down", [False, True])
def test_zeros_before_the_tokens(dtype, down):
    x, dt, a, b, c = _inputs(dtype, down)
    x[:, :-TAIL] = 0
    x = x * 2.0 ** -14  # (64 tokens grow a state by up to e^48)
    b = b * 2.0 ** -14
    y, final = F.selective_scan(x, dt, a, b, c)
    cut = slice(L - TAIL, None)
    part, last = F.selective_scan(x[:, cut], dt[:, cut], a, b[:, cut], c[:, cut])
    assert not y[:, :-TAIL].any()
    assert torch.equal(y[:, cut], part) and torch.equal(final, last)
    assert torch.isfinite(final).all() and final.any()


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("down", [False, True])
def test_gradients_before_a_stretch_of_zeros(dtype, down):
    x, dt, a, b, c = _inputs(dtype, down)
    head = slice(0, 8)
    x = torch.zeros_like(x)
    dy = torch.zeros_like(x)
    dy[:, head] = torch.randn(1, 8, D, device=DEV).to(dtype) / 64

    def gradients(cut):
        leaves = [t[:, cut].clone().requires_grad_() for t in (x, dt, b, c)]
        y, _ = F.selective_scan(leaves[0], leaves[1], a, leaves[2], leaves[3])
        return torch.autograd.grad(y, leaves, dy[:, cut])

    whole, part = gradients(slice(None)), gradients(head)
    for g, p in zip(whole, part):
        assert torch.isfinite(g).all()
        assert torch.equal(g[:, head], p) and not g[:, 8:].any()
    assert part[0].any()
