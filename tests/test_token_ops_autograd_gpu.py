"""How layer norm, linear attention and its single-token form stand with autograd."""

import pytest
import torch
from torch.autograd import forward_ad

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


def test_forward_mode_is_refused():
    """There is no forward-mode derivative: a dual tensor raises, it does not lose its tangent."""
    x, w = torch.randn(4, 16, device=DEV), torch.randn(16, device=DEV)
    q, k, v, a = _tokens()
    state = torch.zeros(2, 2, 16, 16, device=DEV)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        F.layer_norm(x, w)  # plain tensors inside a level are as ever
        F.linear_attention(q, k, v, a, initial_state=state)
        for call in (lambda: F.layer_norm(dual(x), w), lambda: F.layer_norm(x, dual(w)),
                     lambda: F.layer_norm(x, w, dual(w)),
                     lambda: F.linear_attention(dual(q), k, v, a),
                     lambda: F.linear_attention(q, dual(k), v, a),
                     lambda: F.linear_attention(q, k, dual(v), a),
                     lambda: F.linear_attention(q, k, v, a, initial_state=dual(state))):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                call()
        with pytest.raises(ValueError, match="log_decay"):
            F.linear_attention(q, k, v, dual(a))
        for at in range(3):
            tokens = [t[:, 0] for t in (q, k, v)]
            tokens[at] = dual(tokens[at])
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                F.linear_attention_step(*tokens, a, state)
        with pytest.raises(RuntimeError, match="no gradient"):
            F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, dual(state))
