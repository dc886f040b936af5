"""DecayTokenMixer on padded batches: what stands after a sequence's tokens reaches nothing, and outputs
there are zero.  Against other padding the same bits; against each sequence alone 1e-4 of the largest
value in fp32 (a thousand roundings of magnitudes near one)."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

from .test_mixer_padding_gpu import DEV, _padded, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_may_hold_anything(dtype):
    torch.manual_seed(0)
    layer = F.DecayTokenMixer(32, num_heads=4, num_kv_heads=2).to(DEV).to(dtype)
    x = torch.randn(4, 50, 32, device=DEV).to(dtype)
    dy = torch.randn(4, 50, 32, device=DEV).to(dtype)
    lengths = torch.tensor([50, 0, 17, -2], device=DEV)
    want = _run(layer, _padded(x, lengths, 0.5), lengths, _padded(dy, lengths, 0.0))
    live = torch.arange(50, device=DEV) < lengths.unsqueeze(-1)
    assert not want[0][~live].any() and not want[2][0][~live].any()
    for value in (float("nan"), float("inf"), 1e30):
        got = _run(layer, _padded(x, lengths, value), lengths.int(), _padded(dy, lengths, value))
        for p, q in zip([got[0], *got[1], *got[2]], [want[0], *want[1], *want[2]]):
            assert torch.isfinite(p).all() and torch.equal(p, q)


def test_a_padded_batch_is_its_sequences():
    torch.manual_seed(1)
    layer = F.DecayTokenMixer(32, num_heads=4, num_kv_heads=2).to(DEV)
    with torch.no_grad():  # (biases that outputs after the lengths would have)
        layer.out_proj.bias.normal_()
    x, dy = torch.randn(3, 40, 32, device=DEV), torch.randn(3, 40, 32, device=DEV)
    lengths = torch.tensor([40, 9, 23], device=DEV)
    y, states, grads = _run(layer, _padded(x, lengths, float("nan")), lengths, dy)
    sums = [torch.zeros_like(p) for p in layer.parameters()]
    near = lambda p, q: float((p - q).abs().max()) <= 1e-4 * max(1.0, float(q.abs().max()))  # noqa: E731
    for i, n in enumerate(lengths.tolist()):
        one, last, g = _run(layer, x[i:i + 1, :n], None, dy[i:i + 1, :n])
        assert near(y[i, :n], one[0]) and near(grads[0][i, :n], g[0][0])
        assert near(states[0][i], last[0][0])
        sums = [s + t for s, t in zip(sums, g[1:])]
    assert all(near(p, q) for p, q in zip(grads[1:], sums))
    with pytest.raises(ValueError, match="lengths"):
        layer(x, lengths=lengths[:1])
