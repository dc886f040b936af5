"""causal_conv1d, its gradients and its single-token form against the formula in 64 bits.

Tolerances, set from the arithmetic: a result rounded once to a type of unit roundoff u is off by
u |result|.  A sum of W taps and a bias in 32 bits is off by (W + 1) 2^-24 of the sum of
magnitudes; silu's slope is at most 1.1, and its sigmoid comes from the exponential (fp32 rows: 2
roundings and a division's; 16-bit rows: the fast ones, 2 + 1.2 |p| and 2 roundings), written here
as ``GROWTH`` = 32 roundings of (1 + |p|) times what enters.  A gradient's sum over N tokens runs
in short runs joined in order: 32 + 48 roundings of the sum of magnitudes.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, F32, F16, BF16 = torch.float64, torch.float32, torch.float16, torch.bfloat16
ROUND = {F64: 2.0 ** -53, F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F64: 1e-300, F32: 2.0 ** -126, F16: 2.0 ** -24, BF16: 2.0 ** -126}
GROWTH = 32


def _acc(dtype):
    return 2.0 ** -53 if dtype == F64 else 2.0 ** -24


def _case(B, L, D, W, dtype, param=None, bias=True, initial=True, lengths=None, seed=0):
    torch.manual_seed(seed)
    x = torch.randn(B, L, D, device=DEV).to(dtype)
    w = torch.randn(D, W, device=DEV).to(param or dtype)
    b = torch.randn(D, device=DEV).to(param or dtype) if bias else None
    i = torch.randn(B, W - 1, D, device=DEV).to(dtype) if initial else None
    n = None if lengths is None else torch.tensor(lengths, device=DEV, dtype=torch.int32)
    return x, w, b, i, n


def _reference(x, w, b, i, n, silu, dy=None, df=None):
    """y, final, and with dy the gradients, with the sums of magnitudes behind each."""
    x, w = x.detach().double(), w.detach().double()
    B, L, D = x.shape
    W = w.shape[1]
    count = torch.full((B,), L, device=DEV) if n is None else n.clamp(0, L).long()
    live = (torch.arange(L, device=DEV) < count.view(B, 1)).unsqueeze(-1)
    line = torch.zeros(B, W - 1 + L, D, device=DEV, dtype=F64)
    if i is not None:
        line[:, :W - 1] = i.detach().double()
    line[:, W - 1:] = torch.where(live, x, 0.0)
    p = torch.zeros(B, L, D, device=DEV, dtype=F64)
    mag = torch.zeros_like(p)
    if b is not None:
        p, mag = p + b.detach().double(), mag + b.detach().double().abs()
    for j in range(W):
        p = p + w[:, j] * line[:, j:j + L]
        mag = mag + (w[:, j] * line[:, j:j + L]).abs()
    s = torch.sigmoid(p)
    y = p * s if silu else p
    slope = s * (1 + p * (1 - s)) if silu else torch.ones_like(p)
    final = torch.stack([line[k, count[k]:count[k] + W - 1] for k in range(B)])
    mag = mag * (1 + p.abs()) if silu else mag
    out = {"y": torch.where(live, y, 0.0), "mag": mag, "final": final}
    if dy is None:
        return out
    dp = torch.where(live, dy.double() * slope, 0.0)
    # a slope's own error: its derivative is at most 1/2, and the sigmoid's roundings
    err = torch.where(live, dy.double().abs() * (1 + mag), 0.0) if silu else dp.abs()
    dline, eline = torch.zeros_like(line), torch.zeros_like(line)
    dw, ew = torch.zeros_like(w), torch.zeros_like(w)
    for j in range(W):
        dline[:, j:j + L] += w[:, j] * dp
        eline[:, j:j + L] += w[:, j].abs() * err
        dw[:, j] = (dp * line[:, j:j + L]).sum((0, 1))
        ew[:, j] = (err * line[:, j:j + L].abs()).sum((0, 1))
    if df is not None:
        for k in range(B):
            dline[k, count[k]:count[k] + W - 1] += df[k].double()
            eline[k, count[k]:count[k] + W - 1] += df[k].double().abs()
    out |= {"x": torch.where(live, dline[:, W - 1:], 0.0), "x_mag": eline[:, W - 1:],
            "i": dline[:, :W - 1], "i_mag": eline[:, :W - 1], "w": dw, "w_mag": ew,
            "b": dp.sum((0, 1)), "b_mag": err.sum((0, 1))}
    return out


def _check(got, ref, mag, dtype, what, acc=None, growth=GROWTH):
    assert got.dtype == dtype and got.shape == ref.shape, what
    bound = ROUND[dtype] * ref.abs() + growth * (acc or _acc(dtype)) * mag + TINY[dtype]
    worst = ((got.double() - ref).abs() / bound).max() if ref.numel() else torch.zeros(())
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


CASES = [  # B, L, D, W, bias, initial, lengths
    (1, 1, 1, 2, True, False, None), (1, 1, 8, 4, True, True, None), (2, 2, 16, 4, False, True, None),
    (3, 5, 24, 8, True, True, [5, 0, 1]), (2, 37, 64, 4, True, False, None),
    (4, 65, 33, 3, True, True, [65, 0, 2, 64]), (2, 300, 130, 5, True, True, [299, 7]),
    (3, 513, 256, 4, True, True, None), (2, 700, 1001, 4, False, False, [700, 650]),
    (1, 5000, 40, 6, True, True, None), (2, 1030, 96, 7, True, False, [-3, 9999]),
    (2, 0, 16, 4, True, True, None)]


@pytest.mark.parametrize("dtype,param", [(F32, F32), (F64, F64), (F16, F16), (BF16, BF16),
                                         (BF16, F32)])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("B,L,D,W,bias,initial,lengths", CASES)
def test_forward_and_gradients(B, L, D, W, bias, initial, lengths, silu, dtype, param):
    x, w, b, i, n = _case(B, L, D, W, dtype, param, bias, initial, lengths, seed=L)
    if n is not None:  # padding may hold anything
        for k, c in enumerate(n.tolist()):
            x[k, max(0, c):] = float("nan")
    leaves = {"x": x, "w": w, "b": b, "i": i}
    leaves = {k: t.requires_grad_() for k, t in leaves.items() if t is not None}
    activation = "silu" if silu else None
    before = _lib.launch_count()
    y, final = F.causal_conv1d(x, w, b, activation, i, n)
    assert _lib.launch_count() > before
    dy = torch.randn(B, L, D, device=DEV).to(dtype)
    df = torch.randn(B, W - 1, D, device=DEV).to(dtype)
    ref = _reference(x, w, b, i, n, silu, dy, df)
    _check(y.detach(), ref["y"], ref["mag"], dtype, "y")
    assert torch.equal(final.detach().double(), ref["final"])
    with torch.no_grad():
        again = F.causal_conv1d(x, w, b, activation, i, n)
    assert torch.equal(again[0], y) and torch.equal(again[1], final)
    grads = dict(zip(leaves, torch.autograd.grad((y, final), list(leaves.values()), (dy, df))))
    for k, g in grads.items():
        kind = param if k in ("w", "b") else dtype
        _check(g, ref[k], ref[k + "_mag"], kind, f"dL/d{k}", _acc(dtype),
               GROWTH + (48 if k in ("w", "b") else 0))


def test_gradients_against_differences():
    """fp64: central differences of step s are off by s^2 / 6 times a third derivative (here below
    100) and 2^-53 / s of the values: 1e-8 of them at s = 1e-5."""
    x, w, b, i, n = _case(2, 6, 3, 4, F64, lengths=[6, 2])
    for t in (x, w, b, i):
        t.requires_grad_()
    for activation in (None, "silu"):
        assert torch.autograd.gradcheck(
            lambda *a: F.causal_conv1d(a[0], a[1], a[2], activation, a[3], n), (x, w, b, i),
            eps=1e-5, atol=1e-7)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_cut_sequence_is_the_whole(dtype):
    """Two calls that hand the state on, or a prompt and single tokens: the same bits as one."""
    x, w, b, i, _ = _case(3, 40, 72, 4, dtype)
    y, final = F.causal_conv1d(x, w, b, "silu", i)
    for cut in (1, 2, 17, 38):
        a, s = F.causal_conv1d(x[:, :cut], w, b, "silu", i)
        c, s = F.causal_conv1d(x[:, cut:], w, b, "silu", s)
        assert torch.equal(torch.cat([a, c], 1), y) and torch.equal(s, final)
    a, s = F.causal_conv1d(x[:, :30], w, b, "silu", i)
    for t in range(30, 40):
        o = F.causal_conv1d_step(x[:, t], w, s, b, "silu")
        assert torch.equal(o, y[:, t])
    assert torch.equal(s, final)


@pytest.mark.parametrize("dtype,param", [(F32, F32), (F64, F64), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("D,W", [(1, 2), (64, 4), (33, 3), (130, 8), (512, 4)])
def test_step_with_slots(D, W, dtype, param):
    x, w, b, _, _ = _case(5, 1, D, W, dtype, param, seed=D)
    pool = torch.randn(7, W - 1, D, device=DEV).to(dtype)
    slots = torch.tensor([6, -1, 0, 7, 3], device=DEV)
    before = pool.clone()
    for activation in (None, "silu"):
        pool.copy_(before)
        y = F.causal_conv1d_step(x[:, 0], w, pool, b, activation, slots)
        want = before.clone()
        for k, slot in enumerate(slots.tolist()):
            if not 0 <= slot < 7:
                assert not y[k].any()
                continue
            ref = _reference(x[k:k + 1], w, b, before[slot:slot + 1], None, activation is not None)
            _check(y[k:k + 1], ref["y"][:, 0], ref["mag"][:, 0], dtype, "y")
            want[slot] = ref["final"][0].to(dtype)
        assert torch.equal(pool, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_offsets(dtype):
    """Inputs that are slices of a projection's result, at any offset, and gradients of them."""
    torch.manual_seed(1)
    wide = torch.randn(2, 50, 200, device=DEV).to(dtype)
    w, b = torch.randn(64, 4, device=DEV).to(dtype), torch.randn(64, device=DEV).to(dtype)
    for begin in (0, 1, 8, 64):
        part = wide[:, :, begin:begin + 64].detach().requires_grad_()
        flat = part.detach().contiguous().requires_grad_()
        dy = torch.randn(2, 64, 50, device=DEV).to(dtype).transpose(1, 2)
        y, f = F.causal_conv1d(part, w, b, "silu")
        yf, ff = F.causal_conv1d(flat, w, b, "silu")
        assert torch.equal(y, yf) and torch.equal(f, ff)
        g, = torch.autograd.grad(y, part, dy)
        gf, = torch.autograd.grad(yf, flat, dy.contiguous())
        assert torch.equal(g, gf)
    rows = wide[:, 0]
    state, other = torch.zeros(2, 3, 64, device=DEV, dtype=dtype), torch.zeros(2, 3, 64, device=DEV, dtype=dtype)
    a = F.causal_conv1d_step(rows[:, 3:67], w, state, b)
    c = F.causal_conv1d_step(rows[:, 3:67].contiguous(), w, other, b)
    assert torch.equal(a, c) and torch.equal(state, other)


def test_non_finite_inputs_reach_their_window_only():
    x, w, b, i, _ = _case(1, 20, 16, 4, F32)
    x[0, 5, 3] = float("nan")
    x[0, 9, 4] = float("inf")
    y, _ = F.causal_conv1d(x, w, b, "silu", i)
    bad = ~torch.isfinite(y)
    assert bad[0, 5:9, 3].all() and not bad[0, :5].any()
    bad[0, 5:9, 3] = False
    bad[0, 9:13, 4] = False
    assert not bad.any()


def test_streams_and_graphs():
    x, w, b, i, _ = _case(2, 200, 64, 4, BF16)
    want = F.causal_conv1d(x, w, b, "silu", i)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.causal_conv1d(x, w, b, "silu", i)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    state = want[1].clone()
    step = lambda s: F.causal_conv1d_step(x[:, 0], w, s, b, "silu")  # noqa: E731
    step(state.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(state)
    other = want[1].clone()
    for _ in range(3):
        graph.replay()
        assert torch.equal(step(other), held) and torch.equal(state, other)


def test_autograd_manners():
    x, w, b, i, _ = _case(2, 9, 16, 4, F32)
    state = i.clone()
    x.requires_grad_()
    y, _ = F.causal_conv1d(x, w, b, "silu", state)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.causal_conv1d_step(x[:, 0], w, state, b)
    with torch.no_grad():
        F.causal_conv1d_step(x[:, 0], w, state, b)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        F.causal_conv1d_step(x[:, 0].detach().clone(), w, i.clone(), b)


def test_refusals():
    x, w, b, i, _ = _case(2, 9, 16, 4, F32)
    with pytest.raises(ValueError, match="B, L, D"):
        F.causal_conv1d(x[0], w, b)
    with pytest.raises(ValueError, match="weight"):
        F.causal_conv1d(x, w[:3], b)
    for taps in (1, 9):
        with pytest.raises(ValueError, match="taps"):
            F.causal_conv1d(x, torch.ones(16, taps, device=DEV))
    with pytest.raises(TypeError, match="weight"):
        F.causal_conv1d(x, w.half())
    with pytest.raises(TypeError, match="one type"):
        F.causal_conv1d(x.half(), w, b.half())
    with pytest.raises(ValueError, match="bias"):
        F.causal_conv1d(x, w, b[:2])
    with pytest.raises(ValueError, match="activation"):
        F.causal_conv1d(x, w, b, "relu")
    with pytest.raises(ValueError, match="state"):
        F.causal_conv1d(x, w, b, None, i[:, :2])
    with pytest.raises(ValueError, match="lengths"):
        F.causal_conv1d(x, w, b, lengths=torch.ones(3, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="B, D"):
        F.causal_conv1d_step(x, w, i, b)
    with pytest.raises(ValueError, match="state"):
        F.causal_conv1d_step(x[:, 0], w, i[:1].clone(), b)
    with pytest.raises(ValueError, match="contiguous"):
        F.causal_conv1d_step(x[:, 0], w, i.transpose(1, 2).contiguous().transpose(1, 2), b)
    with pytest.raises(RuntimeError, match="devices|CUDA"):
        F.causal_conv1d(x, w.cpu(), b)
    with pytest.raises(TypeError):
        F.causal_conv1d(x.int(), w)
