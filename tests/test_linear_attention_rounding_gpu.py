"""What linear_attention rounds: 16-bit results are those of the operator in 32 bits, rounded once.

Against the closed form in 64 bits the root mean square error may then be that of rounding the
64-bit result to the type, e0 (0.3 to 0.4 unit roundoffs u of the result), and little more: the
products take scores, states and weighted values in at least two 16-bit parts, u^2 of a term each
(2^-16 for bf16, 1 % of e0; 2^-22 for fp16), and sum in 32 bits.  These are independent of e0, so
1.05 e0 leaves room for them; one more value rounded to 16 bits would come to 1.2 e0 or more.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from .test_linear_attention_gpu import DEV, _inputs, _reference

pytestmark = pytest.mark.gpu

CASES = [  # B, L, H, Hkv, Dk, Dv, initial, lengths, fast decay
    (2, 300, 4, 4, 64, 64, True, None, False),
    (1, 1100, 2, 2, 128, 128, True, [1030], False),
    (2, 700, 4, 2, 128, 72, True, [700, 259], False),
    (3, 385, 4, 1, 40, 128, False, [385, 130, 0], False),
    (2, 640, 3, 3, 64, 64, True, None, True),
    (1, 2050, 1, 1, 128, 64, False, None, False),
    (8, 129, 8, 8, 16, 32, True, None, False),
    (4, 1, 8, 8, 64, 64, True, None, False),
    (1, 37, 4, 4, 64, 64, False, None, False),
    (2, 64, 4, 2, 128, 64, True, None, False),
    (2, 100, 2, 2, 64, 128, False, [100, 63], False),
]


def _rms(x):
    return x.double().square().mean().sqrt()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,Hk,Dk,Dv,initial,lengths,fast", CASES)
def test_one_rounding(B, L, H, Hk, Dk, Dv, initial, lengths, fast, dtype):
    q, k, v, a, s0, n = _inputs(B, L, H, Hk, Dk, Dv, dtype, L, initial, lengths, fast)
    torch.manual_seed(L + 1)
    do = torch.randn(B, L, H, Dv, device=DEV).to(dtype)
    wrt = [t.requires_grad_() for t in (q, k, v)]
    out, _ = F.linear_attention(q, k, v, a, initial_state=s0, lengths=n)
    got = (out, *torch.autograd.grad(out, wrt, do))
    leaves = [t.detach().double().requires_grad_() for t in wrt]
    ref, _ = _reference(*leaves, a, s0, n, Dk ** -0.5)
    want = (ref.detach(), *torch.autograd.grad(ref, leaves, do.double()))
    for name, g, r in zip(("out", "dq", "dk", "dv"), got, want):
        once = _rms(r.to(dtype).double() - r)
        off = _rms(g.double() - r)
        assert off <= 1.05 * once, f"{name}: {off / once:.3f} times the rounding of the result"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L", [1, 40, 64, 65, 100, 128])
def test_a_sequence_alone_and_in_a_batch(L, dtype):
    """The kernel goes by a sequence's own sizes: up to a chunk of tokens, which is never cut into
    segments, the bits are the same whatever else is in the call."""
    q, k, v, a, s0, _ = _inputs(7, L, 4, 2, 64, 64, dtype, L, True)
    do = torch.randn(7, L, 4, 64, device=DEV).to(dtype)

    def results(rows):
        ts = [t[rows].detach().requires_grad_() for t in (q, k, v, s0)]
        out, final = F.linear_attention(*ts[:3], a, initial_state=ts[3])
        return (out, final, *torch.autograd.grad(out, ts, do[rows]))

    batch = results(slice(0, 7))
    for b in (0, 6):
        for alone, whole in zip(results(slice(b, b + 1)), batch):
            assert torch.equal(alone[0], whole[b])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L", [129, 700])
def test_a_long_sequence_alone_and_in_a_batch(L, dtype):
    """Longer ones are cut into as many segments as the call's blocks leave room for, which adds
    up the same 32-bit sums in another order: (64 + 64 + 128 + L / 32) 2^-24 of their magnitudes
    at most, and 16-bit results a rounding (u of the result) where that decides one."""
    q, k, v, a, s0, _ = _inputs(24, L, 8, 8, 64, 64, dtype, L, True)
    unit = {torch.float32: 0.0, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[dtype]
    with torch.no_grad():
        batch = F.linear_attention(q, k, v, a, initial_state=s0)
        alone = F.linear_attention(q[5:6], k[5:6], v[5:6], a, initial_state=s0[5:6])
        size = _reference(q[5:6].abs(), k[5:6].abs(), v[5:6].abs(), a, s0[5:6].abs(), None, 0.125)
        growth = (256 + L / 32) * 2.0 ** -24
        low = 0.0 if dtype == torch.float32 else 2.0 ** -16  # parts of scores and states
        for one, all_, mag, u in zip(alone, batch, size, (unit, 0.0)):
            one, whole = one[0].double(), all_[5].double()
            assert ((one - whole).abs() <= (growth + (low if u else 0.0)) * mag[0]
                    + u * one.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,Hk,Dk,Dv,lengths", [
    (2, 37, 2, 2, 64, 64, None), (1, 128, 4, 2, 128, 128, None), (3, 200, 2, 1, 48, 80, [200, 77, 1]),
    (2, 300, 2, 2, 128, 64, None), (1, 600, 1, 1, 64, 64, None)])
def test_states_of_16_bit_inputs_keep_32_bits(B, L, H, Hk, Dk, Dv, lengths, dtype):
    """Last states and the initial states' gradients: two fp16 parts of a value leave 2^-22 of it
    out, three bf16 parts less; the matrix unit cuts its 32-bit sum off at each of the L / 16 steps,
    2^-25 of it on average, and 2^-22 covers the sums outside.  Two bf16 parts would leave 2^-19."""
    q, k, v, a, s0, n = _inputs(B, L, H, Hk, Dk, Dv, dtype, L, True, lengths)
    do = torch.randn(B, L, H, Dv, device=DEV).to(dtype)
    ds = torch.randn(B, H, Dk, Dv, device=DEV)
    start = s0.clone().requires_grad_()
    out, final = F.linear_attention(q, k, v, a, initial_state=start, lengths=n)
    (ds0,) = torch.autograd.grad((out, final), start, (do, ds))
    rstart = s0.double().requires_grad_()
    rout, rfinal = _reference(q, k, v, a, rstart, n, Dk ** -0.5)
    (rds0,) = torch.autograd.grad((rout, rfinal), rstart, (do.double(), ds.double()))
    bound = 2.0 ** -21 + L / 16 * 2.0 ** -25
    for name, got, ref in (("final state", final, rfinal), ("ds0", ds0, rds0)):
        off = _rms(got.double() - ref) / _rms(ref)
        assert off <= bound, f"{name}: {off:.3g}, bound {bound:.3g}"
