"""The bounded waits of the tensor-core linear attention, made to run out on purpose.

``fdwt_set_copy_wait_test`` makes block 0 expect 16 bytes more than its first copy brings: every
issued copy still lands, and the wait for the others runs out.  All warps of the block must then
leave their loops, the products and copies in flight end, and the error word read 1, with the
context usable.  Nothing here faults: the only thing changed is the byte count a wait expects.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib, config

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,length", [(64, 300), (128, 700), (64, 9000)])
def test_wait_that_runs_out_sets_the_error_word(dtype, D, length):
    torch.manual_seed(5)
    q, k, v = (torch.randn(1, length, 2, D, device=DEV).to(dtype) for _ in range(3))
    a = torch.tensor([-0.01, -0.1], device=DEV)
    want, state = F.linear_attention(q, k, v, a)
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
    _lib.set_copy_wait_test(16)
    try:
        F.linear_attention(q, k, v, a)
        torch.cuda.synchronize()
    finally:
        _lib.set_copy_wait_test(0, 0)
    assert _lib.device_error() == 1  # a block gave up and returned
    assert _lib.device_error() == 0  # reading clears the word
    again, other = F.linear_attention(q, k, v, a)
    assert torch.equal(again, want) and torch.equal(other, state)
    assert _lib.device_error() == 0


def test_checked_call_raises():
    q, k, v = (torch.randn(1, 300, 1, 64, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    a = torch.tensor([-0.01], device=DEV)
    config.check_device_errors = True
    _lib.set_copy_wait_test(16)
    try:
        with pytest.raises(RuntimeError, match="linattn"):
            F.linear_attention(q, k, v, a)
        _lib.set_copy_wait_test(0, 0)
        F.linear_attention(q, k, v, a)
    finally:
        _lib.set_copy_wait_test(0, 0)
        config.check_device_errors = False


def test_many_sequences_and_heads():
    """More sequences times heads than one axis of a grid holds."""
    B, H, D = 8200, 16, 16
    torch.manual_seed(6)
    q, k, v = (torch.randn(B, 66, H, D, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    a = -torch.linspace(0.01, 0.5, H, device=DEV)
    out, state = F.linear_attention(q, k, v, a)
    part = slice(B - 40, B)
    ref, last = F.linear_attention(q[part].float(), k[part].float(), v[part].float(), a)
    # scores, the state's copy and the result rounded once each (unit roundoff 2^-8)
    assert (out[part].float() - ref).square().mean().sqrt() <= 2 * 2.0 ** -8 * ref.square().mean().sqrt()
    assert (state[part] - last).abs().max() <= 1e-4 * last.abs().max()


@pytest.mark.parametrize("word", [0xFFFFFFFF, 0x7F800000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length,Dk,Dv", [(70, 24, 40), (1500, 128, 72), (3000, 64, 64)])
def test_nothing_depends_on_what_shared_memory_held(length, Dk, Dv, dtype, word):
    """With all of shared memory set to NaN (infinity) before every kernel the results keep their
    bits: forward, gradients, a token, and the norm."""
    torch.manual_seed(7)
    q = torch.randn(2, length, 2, Dk, device=DEV).to(dtype)
    k = torch.randn(2, length, 1, Dk, device=DEV).to(dtype)
    v = torch.randn(2, length, 1, Dv, device=DEV).to(dtype)
    do = torch.randn(2, length, 2, Dv, device=DEV).to(dtype)
    a = torch.tensor([-0.3, -0.002], device=DEV)
    n = torch.tensor([length, length // 3], device=DEV)
    x, w = do.reshape(-1, 2 * Dv), torch.randn(2 * Dv, device=DEV).to(dtype)

    def everything():
        ts = [t.detach().requires_grad_() for t in (q, k, v)]
        out, state = F.linear_attention(*ts, a, lengths=n)
        results = [out, state, *torch.autograd.grad(out, ts, do)]
        carried = state.detach().clone()
        results += [F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, carried), carried]
        ps = [t.detach().requires_grad_() for t in (x, w)]
        y = F.layer_norm(*ps)
        return results + [y, *torch.autograd.grad(y, ps, y.detach())]

    want = everything()
    _lib.set_shared_memory_fill(True, word)
    try:
        got = everything()
        torch.cuda.synchronize()
    finally:
        _lib.set_shared_memory_fill(False)
    for g, r in zip(got, want):
        assert torch.equal(g, r)
