"""What linear_attention keeps between calls: descriptors of types, sizes, strides and scale."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200.linear_attention import _SEQUENCE, _plan


def test_scale_is_taken_by_value():
    """A scale held in a tensor or an array that changes in place between calls."""
    q = torch.zeros(1, 8, 2, 16)
    scale = torch.tensor(0.5)
    assert _plan(_SEQUENCE, q, q, q, scale)[0].scale == 0.5
    scale.fill_(0.25)
    assert _plan(_SEQUENCE, q, q, q, scale)[0].scale == 0.25
    assert _plan(_SEQUENCE, q, q, q, scale.double().numpy())[0].scale == 0.25
    assert _plan(_SEQUENCE, q, q, q, 2)[0].scale == 2.0
    assert _plan(_SEQUENCE, q, q, q, None)[0].scale == 0.25
    with pytest.raises(ValueError, match="gradient"):
        _plan(_SEQUENCE, q, q, q, torch.tensor(0.5, requires_grad=True))


@pytest.mark.gpu
def test_backward_keeps_the_scale_of_its_forward():
    """Also where d_out has strides of its own, for which the backward pass plans anew."""
    torch.manual_seed(0)
    q, k, v = (torch.randn(1, 20, 2, 16, device="cuda") for _ in range(3))
    a = torch.tensor([-0.1, -0.2], device="cuda")
    scale = torch.tensor(0.5)
    q.requires_grad_()
    (want,) = torch.autograd.grad(F.linear_attention(q, k, v, a, scale=0.5)[0].sum(), q)
    out, _ = F.linear_attention(q, k, v, a, scale=scale)
    scale.fill_(2.0)
    (got,) = torch.autograd.grad(out.sum(), q)
    assert torch.equal(got, want)
