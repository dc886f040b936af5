"""The causal mixers on padded batches: what stands after a sequence's tokens, in the inputs and in the
gradients of the outputs, reaches nothing, and outputs there are zero.  Against other padding: the same
bits.  Against each sequence alone, in fp32: 1e-4 of the largest value, as the layers' other tests
(some thousand roundings of magnitudes near one)."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
LAYERS = {
    "mixer": lambda: F.SelectiveTokenMixer(32, state_size=8),
    "stack": lambda: F.SelectiveTokenStack(32, 2, state_size=5),
}


def _flat(state):
    return [state] if isinstance(state, torch.Tensor) else [t for s in state for t in _flat(s)]


def _run(layer, x, lengths, dy):
    x = x.detach().clone().requires_grad_()
    y, state = layer(x, lengths=lengths, return_state=True)
    outs = [y, *_flat(state)]
    grads = torch.autograd.grad(outs, [x, *layer.parameters()],
                                [dy, *(torch.ones_like(t) for t in outs[1:])])
    return y.detach(), [t.detach() for t in outs[1:]], grads


def _padded(t, lengths, value):
    t = t.clone()
    for i, n in enumerate(lengths.tolist()):
        t[i, max(0, n):] = value
    return t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", LAYERS)
def test_padding_may_hold_anything(kind, dtype):
    torch.manual_seed(0)
    layer = LAYERS[kind]().to(DEV).to(dtype)
    x = torch.randn(4, 50, 32, device=DEV).to(dtype)
    dy = torch.randn(4, 50, 32, device=DEV).to(dtype)
    lengths = torch.tensor([50, 0, 17, -2], device=DEV)
    want = _run(layer, _padded(x, lengths, 0.5), lengths, _padded(dy, lengths, 0.0))
    live = torch.arange(50, device=DEV) < lengths.unsqueeze(-1)
    assert not want[0][~live].any() and not want[2][0][~live].any()
    for value in (float("nan"), float("inf"), 1e30):
        for n in (lengths, lengths.int()):
            got = _run(layer, _padded(x, lengths, value), n, _padded(dy, lengths, value))
            assert torch.equal(got[0], want[0])
            for p, q in zip([*got[1], *got[2]], [*want[1], *want[2]]):
                assert torch.isfinite(p).all() and torch.equal(p, q)


@pytest.mark.parametrize("kind", LAYERS)
def test_a_padded_batch_is_its_sequences(kind):
    torch.manual_seed(1)
    layer = LAYERS[kind]().to(DEV)
    x, dy = torch.randn(3, 40, 32, device=DEV), torch.randn(3, 40, 32, device=DEV)
    lengths = torch.tensor([40, 9, 23], device=DEV)
    y, states, grads = _run(layer, _padded(x, lengths, float("nan")), lengths, dy)
    sums = [torch.zeros_like(p) for p in layer.parameters()]
    near = lambda p, q: float((p - q).abs().max()) <= 1e-4 * max(1.0, float(q.abs().max()))  # noqa: E731
    for i, n in enumerate(lengths.tolist()):
        one, last, g = _run(layer, x[i:i + 1, :n], None, dy[i:i + 1, :n])
        assert near(y[i, :n], one[0]) and near(grads[0][i, :n], g[0][0])
        assert all(near(s[i], t[0]) for s, t in zip(states, last))
        sums = [s + t for s, t in zip(sums, g[1:])]
    assert all(near(p, q) for p, q in zip(grads[1:], sums))


@pytest.mark.parametrize("kind", LAYERS)
def test_lengths_of_another_shape_or_type_are_refused(kind):
    layer = LAYERS[kind]().to(DEV)
    x = torch.randn(2, 5, 32, device=DEV)
    for bad in (torch.ones(3, device=DEV, dtype=torch.int32), torch.ones(1, device=DEV, dtype=torch.int32),
                torch.ones(2, device=DEV), torch.ones(2, 1, device=DEV, dtype=torch.int64)):
        with pytest.raises(ValueError, match="lengths"):
            layer(x, lengths=bad)
