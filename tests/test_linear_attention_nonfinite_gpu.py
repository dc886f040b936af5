"""Infinities and NaN in linear_attention stay where the recurrence takes them.

    S_t = d S_{t-1} + k_t v_t^T,   o_t = scale q_t^T S_t

A non-finite v_s[c] makes column c of the states and outputs non-finite from token s on, a
non-finite k_s whole outputs from s on, a non-finite q_t the output t alone.  Backward in time the
same holds for dL/do and q.  Everything else keeps its bits, or where it is formed in another order
of 32-bit sums its value (the other columns after s; in 16 bits column c before s): a 16-bit
result may then round the other way, u of it and 2^-12 of the largest at most.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.float64: 2.0 ** -48, torch.float32: 2.0 ** -20, torch.float16: 2.0 ** -10,
        torch.bfloat16: 2.0 ** -7}


def _everything(q, k, v, do, a, s0):
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    out, final = F.linear_attention(*leaves[:3], a, initial_state=leaves[3])
    return dict(zip(("out", "final", "dq", "dk", "dv", "ds0"),
                    (out.detach(), final.detach(), *torch.autograd.grad(out, leaves, do))))


def _close(x, y, dtype):
    x, y = x.double(), y.double()
    assert x.isfinite().all()
    most = y.abs().max() if y.numel() else 0.0
    assert ((x - y).abs() <= UNIT[dtype] * y.abs() + 2.0 ** -12 * most).all()


CASES = [(torch.float32, 64, 48), (torch.float32, 128, 96), (torch.float32, 200, 40),
         (torch.float64, 24, 40), (torch.float64, 160, 160), (torch.bfloat16, 64, 64),
         (torch.bfloat16, 128, 80), (torch.float16, 64, 64), (torch.float16, 128, 80),
         (torch.bfloat16, 20, 28), (torch.float16, 100, 33)]


@pytest.mark.parametrize("dtype,Dk,Dv", CASES)
@pytest.mark.parametrize("at", [0, 5, 70, 127, 128, 299])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_value_reaches_no_token_that_does_not_depend_on_it(dtype, Dk, Dv, at, value):
    torch.manual_seed(at + Dk)
    B, L, H = 2, 300, 2
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    q, k = (torch.randn(B, L, H, Dk, device=DEV).to(dtype) for _ in range(2))
    v, do = (torch.randn(B, L, H, Dv, device=DEV).to(dtype) for _ in range(2))
    s0 = torch.randn(B, H, Dk, Dv, device=DEV, dtype=acc)
    a = torch.tensor([-0.02, -0.001], device=DEV, dtype=acc)
    clean = _everything(q, k, v, do, a, s0)
    before, own, after = slice(0, at), slice(at, at + 1), slice(at + 1, L)
    upto, since = slice(0, at + 1), slice(at, L)
    col = Dv // 2 + 3
    dim = Dk // 2 + 3
    b, h = 1, 0

    def check(got, same, gone, columns):
        """same: (result, tokens[, column that may be formed anew]) that keep their bits; gone:
        (result, tokens) of which nothing is finite; columns: (result, tokens, column) where only
        that column is not finite."""
        for name in clean:  # the other sequence and the other head
            x, y = got[name], clean[name]
            assert torch.equal(x[0], y[0])
            if name in ("final", "ds0"):
                assert torch.equal(x[b, 1], y[b, 1])
            else:
                assert torch.equal(x[b, :, 1], y[b, :, 1])
        for name, t, *anew in same:
            x, y = got[name][b, t, h], clean[name][b, t, h]
            if anew and dtype.itemsize == 2:
                _close(x[:, anew[0]], y[:, anew[0]], dtype)
                keep = [i for i in range(x.shape[1]) if i != anew[0]]
                x, y = x[:, keep], y[:, keep]
            assert torch.equal(x, y), name
        for name, t in gone:
            assert not got[name][b, t, h].isfinite().any(), name
        for name, t, c in columns:
            x, y = got[name][b, t, h], clean[name][b, t, h]
            assert not x[:, c].isfinite().any(), name
            keep = [i for i in range(x.shape[1]) if i != c]
            _close(x[:, keep], y[:, keep], dtype)

    whole = slice(0, L)
    bad = v.clone()
    bad[b, at, h, col] = value
    got = _everything(q, k, bad, do, a, s0)
    check(got, [("out", before, col), ("dq", before), ("dk", before), ("dk", after),
                ("dv", whole)],
          [("dq", since), ("dk", own)], [("out", since, col)])
    assert torch.equal(got["ds0"], clean["ds0"])
    assert not got["final"][b, h, :, col].isfinite().any()
    keep = [i for i in range(Dv) if i != col]
    _close(got["final"][b, h][:, keep], clean["final"][b, h][:, keep], dtype)

    bad = k.clone()
    bad[b, at, h, dim] = value
    got = _everything(q, bad, v, do, a, s0)
    check(got, [("out", before), ("dq", before, dim), ("dv", before), ("dv", after),
                ("dk", whole)],
          [("out", since), ("dv", own)], [("dq", since, dim)])
    assert torch.equal(got["ds0"], clean["ds0"])

    bad = q.clone()
    bad[b, at, h, dim] = value
    got = _everything(bad, k, v, do, a, s0)
    check(got, [("out", before), ("out", after), ("dq", whole), ("dk", after, dim),
                ("dv", after)],
          [("out", own), ("dv", upto)], [("dk", upto, dim)])
    assert torch.equal(got["final"], clean["final"])

    bad = do.clone()
    bad[b, at, h, col] = value
    got = _everything(q, k, v, bad, a, s0)
    check(got, [("out", whole), ("dq", before), ("dq", after), ("dk", after),
                ("dv", after, col)],
          [("dq", own), ("dk", upto)], [("dv", upto, col)])


@pytest.mark.parametrize("L", [700, 3000, 9000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_many_values(dtype, L):
    """Several tokens and columns of a chunk, and of other chunks and segments."""
    torch.manual_seed(3)
    D = 64
    q, k, v = (torch.randn(1, L, 1, D, device=DEV).to(dtype) for _ in range(3))
    a = torch.tensor([-0.01], device=DEV)
    clean, _ = F.linear_attention(q, k, v, a)
    first = torch.full((D,), L, device=DEV)
    for t, c in [(130, 0), (131, 0), (140, 1), (135, 1), (200, 63), (260, 9), (390, 10), (699, 11),
                 (698, 12), (256, 13), (511, 14), (512, 15), (640, 1), (L // 2 + 3, 20),
                 (L - 130, 21), (L - 1, 22)]:
        v[0, t, 0, c] = float("nan") if t % 2 else float("inf")
        first[c] = min(int(first[c]), t)
    out, final = F.linear_attention(q, k, v, a)
    reached = torch.arange(L, device=DEV).view(L, 1) >= first
    assert torch.equal(out[0, :, 0].isfinite(), ~reached)
    assert torch.equal(final[0, 0].isfinite().all(0), first == L)
    keep = ~reached
    _close(out[0, :, 0][keep], clean[0, :, 0][keep], dtype)


@pytest.mark.parametrize("dtype,Dk,Dv", CASES)
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_an_initial_state_that_is_not_finite(dtype, Dk, Dv, value):
    """It passes through a sequence without tokens as it is, and stays in its column of another."""
    torch.manual_seed(Dk)
    L, H = 200, 2
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    q, k = (torch.randn(2, L, H, Dk, device=DEV).to(dtype) for _ in range(2))
    v = torch.randn(2, L, H, Dv, device=DEV).to(dtype)
    s0 = torch.randn(2, H, Dk, Dv, device=DEV, dtype=acc)
    a = torch.tensor([-0.02, -0.001], device=DEV, dtype=acc)
    n = torch.tensor([0, L], device=DEV)
    clean, last = F.linear_attention(q, k, v, a, initial_state=s0, lengths=n)
    s0[:, 0, Dk // 2, Dv // 2] = value
    out, final = F.linear_attention(q, k, v, a, initial_state=s0, lengths=n)
    assert torch.equal(final[0].nan_to_num(7.0), s0[0].nan_to_num(7.0)) and not out[0].any()
    keep = [i for i in range(Dv) if i != Dv // 2]
    assert torch.equal(out[1, :, 1], clean[1, :, 1]) and torch.equal(final[1, 1], last[1, 1])
    assert not out[1, :, 0, Dv // 2].isfinite().any()
    # the entry itself: times the decay it is what it was
    got = final[1, 0, Dk // 2, Dv // 2]
    assert got.isnan() if value != value else got == value
    _close(out[1, :, 0][:, keep], clean[1, :, 0][:, keep], dtype)
    _close(final[1, 0][:, keep], last[1, 0][:, keep], dtype)
