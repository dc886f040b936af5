"""causal_conv1d's gradients where a window holds an infinity or NaN that they do not depend on: the
state of an empty sequence, and last inputs that only some of the taps meet.  What is independent of a
value is the same bit by bit whatever it is."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

from .test_causal_conv_gpu import BF16, DEV, F16, F32, F64, _case

pytestmark = pytest.mark.gpu
DTYPES = [F32, F64, F16, BF16]


def _gradients(x, w, b, i, n, activation, dy, df):
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, i)]
    y, final = F.causal_conv1d(leaves[0], leaves[1], leaves[2], activation, leaves[3], n)
    return torch.autograd.grad((y, final), leaves, (dy, df))


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,D,W", [(9, 16, 4), (70, 33, 8), (300, 64, 2), (0, 8, 3)])
def test_the_state_of_an_empty_sequence(L, D, W, dtype, activation):
    """Its gradient is the final state's, and nothing else meets it."""
    x, w, b, i, _ = _case(3, L, D, W, dtype, seed=D)
    n = torch.tensor([L, 0, max(0, L - 3)], device=DEV, dtype=torch.int32)
    dy = torch.randn(3, L, D, device=DEV).to(dtype)
    df = torch.randn(3, W - 1, D, device=DEV).to(dtype)
    want = _gradients(x, w, b, i, n, activation, dy, df)
    for bad in (float("nan"), float("inf")):
        state = i.clone()
        state[1] = bad
        got = _gradients(x, w, b, state, n, activation, dy, df)
        assert all(torch.isfinite(g).all() for g in got)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert torch.equal(got[3][1], df[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,D,W,count", [(9, 16, 4, 9), (70, 33, 8, 61), (300, 64, 3, 300), (64, 40, 4, 64)])
def test_last_inputs_meet_only_their_taps(L, D, W, count, dtype):
    """Input count - 1 - k, k < W - 1, has products with the last k + 1 taps' gradients alone (no
    activation: the slope is 1)."""
    x, w, b, i, _ = _case(2, L, D, W, dtype, seed=L)
    n = torch.tensor([count, L], device=DEV, dtype=torch.int32)
    dy = torch.randn(2, L, D, device=DEV).to(dtype)
    df = torch.randn(2, W - 1, D, device=DEV).to(dtype)
    want = _gradients(x, w, b, i, n, None, dy, df)
    for k in range(W - 1):
        bad = x.clone()
        bad[0, count - 1 - k, 3] = float("nan")
        bad[0, count - 1 - k, 5] = float("inf")
        got = _gradients(bad, w, b, i, n, None, dy, df)
        for c in (3, 5):
            assert torch.equal(got[1][c, :W - 1 - k], want[1][c, :W - 1 - k])
            assert not torch.isfinite(got[1][c, W - 1 - k:]).any()
        keep = [c for c in range(D) if c not in (3, 5)]
        assert torch.equal(got[1][keep], want[1][keep])
        assert all(torch.equal(got[j], want[j]) for j in (0, 2, 3))
