"""How layer norm, linear attention and its single-token form stand with autograd."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tokens(L=20, H=2, D=16, dtype=torch.float32):
    torch.manual_seed(L)
    q, k, v = (torch.randn(2, L, H, D, device=DEV, dtype=dtype) for _ in range(3))
    return q, k, v, torch.tensor([-0.1] * H, device=DEV)


@pytest.mark.parametrize("use_slots", [False, True])
def test_step_counts_as_a_change_of_the_state(use_slots):
    """A state that an earlier call saved and a step then overwrote: its backward pass raises."""
    q, k, v, a = _tokens()
    state = torch.randn(2, 2, 16, 16, device=DEV)
    slots = torch.tensor([1, 0], device=DEV) if use_slots else None
    q.requires_grad_()
    out, _ = F.linear_attention(q, k, v, a, initial_state=state)
    before = state._version
    with torch.no_grad():
        F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, state, slots=slots)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_step_on_inference_states():
    q, k, v, a = _tokens()
    with torch.inference_mode():
        state = torch.zeros(2, 2, 16, 16, device=DEV)
        out = F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, state)
    plain = torch.zeros(2, 2, 16, 16, device=DEV)
    assert torch.equal(out, F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, plain))
    assert torch.equal(state, plain)
