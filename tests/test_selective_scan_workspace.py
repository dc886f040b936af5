"""The workspace of the scan's backward pass: its bound, and calls whose parts of dL/db and dL/dc do not
fit it at once.

Where nothing is remembered (rates of -inf) and inputs are small whole numbers, every gradient is a sum
of whole numbers, exact in 32 bits in any order: dL/db_t[n] = c_t[n] sum_d dy x, dL/dc_t[n] = b_t[n]
sum_d dy x, dL/dx = dy <c, b>, dL/ddt = x dL/dx (steps of 1).  16-bit results are those rounded once."""

import ctypes

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

from .test_selective_ops_host import PTR, WORKSPACE, _scan

DEV = "cuda"
F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16
GIB = 1 << 30


def test_the_workspace_is_bounded():
    lib = _lib.load()
    for dtype in (0, 1, 3):
        for states in (1, 5, 16, 33, 64, 128):
            for groups in (1, 2, 16):
                for batch, length in ((1, 65536), (4, 4096), (64, 1024), (3, 100), (2, 0)):
                    at = _scan(dtype, groups, states, batch, length, 2048)
                    d = ctypes.addressof(at)
                    size = 8 if dtype == 1 else 4
                    padded = max(4, 1 << (states - 1).bit_length())
                    tile = batch * length * 2 * padded * size
                    least = lib.fdwt_selscan_backward_workspace_least(d)
                    need = lib.fdwt_selscan_backward_workspace(d)
                    # sums of da, dskip and dt_bias, and states between segments, for each of up to 64
                    assert least <= batch * 64 * 2048 * (2 * padded + 3) * size + 1024
                    assert least <= need <= least + max(GIB, tile) + groups * tile + 512
    # 65536 tokens of 2048 channels: 17 GB with all parts at once
    assert lib.fdwt_selscan_backward_workspace(
        ctypes.addressof(_scan(3, 1, 128, 1, 65536, 2048))) < 1.4e9


def test_the_least_workspace_is_enough_without_b_and_c():
    lib = _lib.load()
    good = _scan()
    at = ctypes.addressof(good)
    least = lib.fdwt_selscan_backward_workspace_least(at)
    need = lib.fdwt_selscan_backward_workspace(at)
    assert 0 < least < need
    call = lambda db, dc, n: lib.fdwt_selscan_backward(  # noqa: E731
        at, *[PTR] * 15, db, dc, *[PTR] * 5, n, None)
    assert call(None, None, least - 1) == WORKSPACE
    for db, dc in ((PTR, None), (None, PTR), (PTR, PTR)):
        assert call(db, dc, need - 1) == WORKSPACE


def _whole_numbers(B, L, D, N, G, dtype):
    torch.manual_seed(D)
    t = lambda *s: torch.randint(-2, 3, s, device=DEV).to(dtype).requires_grad_()  # noqa: E731
    x, b, c = t(B, L, D), t(B, L, G, N), t(B, L, G, N)
    dt = torch.ones_like(x).requires_grad_()
    wide = F64 if dtype == F64 else F32
    a = torch.full((D, N), float("-inf"), device=DEV, dtype=wide)
    return x, dt, a, b, c, t(B, L, D).detach()


def _check(x, dt, a, b, c, dy, lengths, leaves=("x", "dt", "b", "c")):
    B, L, D = x.shape
    G = b.shape[2]
    y, _ = F.selective_scan(x, dt, a, b, c, lengths=lengths)
    named = {"x": x, "dt": dt, "b": b, "c": c}
    got = dict(zip(leaves, torch.autograd.grad(y, [named[k] for k in leaves], dy)))
    live = torch.ones(B, L, 1, device=DEV, dtype=F64)
    if lengths is not None:
        live = (torch.arange(L, device=DEV) < lengths.unsqueeze(-1)).unsqueeze(-1).double()
    xd, bd, cd, q = (t.detach().double() for t in (x, b, c, dy))
    met = (q * xd * live).unflatten(-1, (G, D // G)).sum(-1, keepdim=True)   # (B, L, G, 1)
    across = (bd * cd).sum(-1).repeat_interleave(D // G, -1) * live
    want = {"b": cd * met, "c": bd * met, "x": q * across, "dt": xd * q * across}
    for k, g in got.items():
        assert torch.equal(g, want[k].to(g.dtype)), k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F64])
def test_parts_in_one_launch(dtype):
    for B, L, D, N, G in ((2, 50, 256, 128, 1), (1, 700, 96, 16, 3), (3, 9, 80, 5, 2)):
        x, dt, a, b, c, dy = _whole_numbers(B, L, D, N, G, dtype)
        lengths = torch.tensor([L, 7, 0][:B], device=DEV, dtype=torch.int32)
        for n in (None, lengths):
            _check(x, dt, a, b, c, dy, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,L,D,N,G", [
    (F32, 1, 36864, 256, 128, 1),     # 32 tiles of 36 MiB: 28 and 4
    (BF16, 2, 18433, 288, 128, 3),    # 36 tiles of 12 a group: 28 and 8, the third group in both
    (F32, 1, 140001, 128, 100, 2),    # 16 tiles of 137 MiB: 7, 7 and 2
    (F64, 1, 20000, 256, 128, 1)])
def test_parts_in_several_launches(dtype, B, L, D, N, G):
    d = _scan(_lib.DTYPES[dtype], G, N, B, L, D)
    at = ctypes.addressof(d)
    lib = _lib.load()
    assert (lib.fdwt_selscan_backward_workspace(at) - lib.fdwt_selscan_backward_workspace_least(at)
            > GIB - 256 * GIB // 1024)  # as many parts at once as fit
    x, dt, a, b, c, dy = _whole_numbers(B, L, D, N, G, dtype)
    _check(x, dt, a, b, c, dy, None)
    lengths = torch.tensor([L - 777, L][:B], device=DEV, dtype=torch.int32)
    _check(x, dt, a, b, c, dy, lengths)
    _check(x, dt, a, b, c, dy, None, ("b",))
    _check(x, dt, a, b, c, dy, None, ("c", "x"))


@pytest.mark.gpu
def test_several_launches_with_a_memory():
    """With states that last, against the halves of the channels in calls of their own, whose parts fit
    at once: gradients of channels side by side, those of b and c added.  fp32: some hundred roundings of
    the largest terms, 1e-4 of the largest value."""
    torch.manual_seed(0)
    L, D, N = 36864, 256, 128
    t = lambda *s: torch.randn(*s, device=DEV).requires_grad_()  # noqa: E731
    x, dt, gate, b, c = t(1, L, D), t(1, L, D), t(1, L, D), t(1, L, 1, N), t(1, L, 1, N)
    a = (-torch.rand(D, N, device=DEV)).requires_grad_()
    skip, dy = t(D), torch.randn(1, L, D, device=DEV)

    def gradients(cut):
        y, _ = F.selective_scan(x[..., cut], dt[..., cut], a[cut], b, c, skip[cut], gate[..., cut],
                                dt_softplus=True)
        return torch.autograd.grad(y, (x, dt, gate, a, skip, b, c), dy[..., cut])

    whole = gradients(slice(None))
    lower, upper = gradients(slice(0, D // 2)), gradients(slice(D // 2, D))
    for p, q, r in zip(whole, lower, upper):
        want = q + r  # (each zero in the other's channels)
        assert float((p - want).abs().max()) <= 1e-4 * float(want.abs().max())


@pytest.mark.gpu
def test_frozen_b_and_c():
    """Neither b nor c wants a gradient: the others are the same bits, from a smaller workspace."""
    torch.manual_seed(1)
    x, dt = (torch.randn(2, 300, 64, device=DEV).requires_grad_() for _ in range(2))
    b, c = (torch.randn(2, 300, 1, 16, device=DEV) for _ in range(2))
    a = (-torch.rand(64, 16, device=DEV)).requires_grad_()
    dy = torch.randn(2, 300, 64, device=DEV)
    frozen = torch.autograd.grad(F.selective_scan(x, dt, a, b, c, dt_softplus=True)[0], (x, dt, a), dy)
    b.requires_grad_()
    free = torch.autograd.grad(F.selective_scan(x, dt, a, b, c, dt_softplus=True)[0], (x, dt, a), dy)
    assert all(torch.equal(p, q) for p, q in zip(frozen, free))
