"""rms_norm (with and without the residual's addition), its gradients, and its result in 8 bits,
against the formula in 64 bits.

Tolerances, set from the arithmetic: a result rounded once to a type of unit roundoff u is off by
u |result|; the sums run in 32 bits (64 for fp64) over trees and short runs, so that a row's mean
square, and with it every value of the row, is off by less than ``GROWTH`` = 48 roundings, relative
to the sum of magnitudes that enters (all of one sign in a mean square).  The sum x + residual is
one rounding by definition, and equal bit by bit.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, F32, F16, BF16 = torch.float64, torch.float32, torch.float16, torch.bfloat16
ROUND = {F64: 2.0 ** -53, F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F64: 0.0, F32: 0.0, F16: 2.0 ** -24, BF16: 0.0}
GROWTH = 48
EPS = 1e-6


def _acc(dtype):
    return 2.0 ** -53 if dtype == F64 else 2.0 ** -24


def _case(rows, dim, dtype, stream=None, param=None, seed=0, residual=True):
    torch.manual_seed(seed)
    x = torch.randn(rows, dim, device=DEV).to(dtype)
    r = (3 * torch.randn(rows, dim, device=DEV)).to(stream or dtype) if residual else None
    w = (1 + 0.2 * torch.randn(dim, device=DEV)).to(param or dtype)
    return x, r, w


def _reference(x, r, w, eps=EPS):
    t = x
    if r is not None:
        wide = F64 if x.dtype == F64 else F32
        t = (x.to(wide) + r.to(wide)).to(r.dtype)
    h = t.double()
    rstd = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    h = h * rstd
    return t, h, rstd, h if w is None else h * w.double()


def _check(got, ref, dtype, spread, what, acc=None):
    bound = ROUND[dtype] * ref.abs() + GROWTH * (acc or _acc(dtype)) * spread + TINY[dtype]
    worst = ((got.double() - ref).abs() / bound.clamp(min=1e-300)).max()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


SHAPES = [(1, 1), (3, 2), (5, 31), (4, 32), (2, 100), (7, 255), (9, 256), (300, 257), (65, 1000),
          (33, 1001), (4, 2048), (3, 4097), (2, 8192), (2, 10001), (2, 16384), (1, 40001)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,param", [(F32, F32), (F64, F64), (F16, F16), (BF16, BF16),
                                         (BF16, F32)])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_forward_and_gradients(rows, dim, dtype, param, residual):
    x, r, w = _case(rows, dim, dtype, None, param, seed=dim, residual=residual)
    leaves = [t.requires_grad_() for t in (x, r, w) if t is not None]
    before = _lib.launch_count()
    out = F.rms_norm(x, w, r, EPS)
    assert _lib.launch_count() > before
    y, total = out if residual else (out, None)
    t, h, rstd, ref = _reference(x.detach(), None if r is None else r.detach(), w.detach())
    if residual:
        assert torch.equal(total, t)
    _check(y.detach(), ref, dtype, ref.abs(), "y")
    dy, dt = torch.randn_like(y), torch.randn_like(y)
    with torch.no_grad():  # without gradients the same bits
        plain = F.rms_norm(x, w, r, EPS)
    assert torch.equal(plain[0] if residual else plain, y)

    grads = torch.autograd.grad(out, leaves, (dy, dt) if residual else dy)
    g = dy.double() * w.detach().double()
    mgh = (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - h * mgh)
    spread = rstd * (g.abs() + h.abs() * (g * h).abs().mean(-1, keepdim=True))
    if residual:
        dx, spread = dx + dt.double(), spread + dt.double().abs()
        _check(grads[1], dx, dtype, spread, "dL/dresidual")
    _check(grads[0], dx, dtype, spread, "dL/dx")
    _check(grads[-1], (dy.double() * h).sum(0), param, (dy.double() * h).abs().sum(0), "dL/dweight",
           _acc(dtype))


@pytest.mark.parametrize("rows,dim", [(5, 31), (9, 256), (33, 1001), (4, 2048), (3, 8192), (2, 20000)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("param", [F32, None])
def test_residual_in_32_bits(rows, dim, dtype, param):
    x, r, w = _case(rows, dim, dtype, F32, param, seed=dim)
    for t in (x, r, w):
        t.requires_grad_()
    y, total = F.rms_norm(x, w, r, EPS)
    t, h, rstd, ref = _reference(x.detach(), r.detach(), w.detach())
    assert total.dtype == F32 and torch.equal(total, t) and y.dtype == dtype
    _check(y.detach(), ref, dtype, ref.abs(), "y")
    dy, dt = torch.randn_like(y), torch.randn_like(total)
    gx, gr, gw = torch.autograd.grad((y, total), (x, r, w), (dy, dt))
    g = dy.double() * w.detach().double()
    dx = rstd * (g - h * (g * h).mean(-1, keepdim=True)) + dt.double()
    spread = rstd * (g.abs() + h.abs() * (g * h).abs().mean(-1, keepdim=True)) + dt.double().abs()
    assert gx.dtype == dtype and gr.dtype == F32
    _check(gx, dx, dtype, spread, "dL/dx")
    _check(gr, dx, F32, spread, "dL/dresidual")
    _check(gw, (dy.double() * h).sum(0), w.dtype, (dy.double() * h).abs().sum(0), "dL/dweight",
           2.0 ** -24)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_fused_is_addition_and_norm(dtype):
    x, r, w = _case(37, 520, dtype)
    y, total = F.rms_norm(x, w, r)
    assert torch.equal(total, x + r) and torch.equal(y, F.rms_norm(x + r, w))


def test_gradients_against_differences():
    """fp64: central differences of step s are off by s^2 / 6 times a third derivative (here below
    100) and 2^-53 / s of the values: 1e-8 of them at s = 1e-5."""
    x, r, w = _case(3, 7, F64)
    for t in (x, r, w):
        t.requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: F.rms_norm(a[0], a[2], a[1]), (x, r, w), eps=1e-5,
                                    atol=1e-7)
    assert torch.autograd.gradcheck(lambda a, b: F.rms_norm(a, b), (x, w), eps=1e-5, atol=1e-7)


def test_only_one_output_used():
    x, r, w = _case(6, 40, F32)
    for t in (x, r, w):
        t.requires_grad_()
    y, total = F.rms_norm(x, w, r)
    d = torch.randn_like(y)
    gx, gr, gw = torch.autograd.grad(total, (x, r, w), d, retain_graph=True)
    assert torch.equal(gx, d) and torch.equal(gr, d) and not gw.any()
    both = torch.autograd.grad((y, total), (x, r), (d, torch.zeros_like(d)), retain_graph=True)
    only = torch.autograd.grad(y, (x, r), d)
    assert all(torch.equal(a, b) for a, b in zip(both, only))


@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("dtype,stream,param", [(F16, F16, F32), (BF16, F32, BF16), (F32, F32, F32),
                                                (BF16, BF16, BF16)])
def test_any_offset(dtype, stream, param, offset):
    """Rows, residuals and weights that begin off 16-byte boundaries."""
    for dim in (130, 256, 1002):
        x, r, w = _case(7, dim, dtype, stream, param, seed=dim)

        def at(t, k):
            flat = torch.empty(t.numel() + k, device=DEV, dtype=t.dtype)
            flat[k:] = t.flatten()
            return flat[k:].view(t.shape)

        for ox, orr, ow in ((offset, 0, 0), (0, offset, 0), (0, 0, offset), (offset,) * 3):
            a, b, c = at(x, ox).requires_grad_(), at(r, orr).requires_grad_(), at(w, ow).requires_grad_()
            y, total = F.rms_norm(a, c, b)
            t, h, rstd, ref = _reference(x, r, w)
            assert torch.equal(total, t)
            _check(y.detach(), ref, dtype, ref.abs(), "y")
            dy, dt = torch.randn_like(y), torch.randn_like(total)
            gx, gr, gw = torch.autograd.grad((y, total), (a, b, c), (dy, dt))
            g = dy.double() * w.double()
            dx = rstd * (g - h * (g * h).mean(-1, keepdim=True)) + dt.double()
            spread = rstd * (g.abs() + h.abs() * (g * h).abs().mean(-1, keepdim=True)) + dt.double().abs()
            _check(gx, dx, dtype, spread, "dL/dx")
            _check(gr, dx, stream, spread, "dL/dresidual", 2.0 ** -24)
            _check(gw, (dy.double() * h).sum(0), param, (dy.double() * h).abs().sum(0), "dL/dw",
                   2.0 ** -24)


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype,stream", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,dim,group", [
    (1, 1, 1), (3, 31, None), (5, 64, 32), (4, 128, 128), (9, 256, 32), (7, 256, 128), (3, 300, 100),
    (2, 384, 96), (11, 1000, 8), (6, 1001, 7), (33, 1024, 64), (4, 2048, 128), (4, 2048, None),
    (3, 8192, 128), (2, 8192, 256), (2, 10001, None), (2, 24576, 128), (1, 30000, None)])
def test_quantized(rows, dim, group, dtype, stream, out):
    """q * scale is off by half a step of its type (e4m3: 2^-4 of the value, at least half the
    smallest subnormal 2^-9; int8: 1/2) times the scale, and the roundings of the norm and the
    division; the scale by the roundings alone."""
    x, r, w = _case(rows, dim, dtype, stream, F32 if dtype == BF16 else dtype, seed=dim)
    x[-1] = 0
    r[-1] = 0
    q, scales, total = F.rms_norm_quantized(x, w, r, EPS, group, out)
    t, _, _, ref = _reference(x, r, w)
    assert torch.equal(total, t)
    assert q.dtype == out and q.shape == x.shape and scales.dtype == F32
    size = group or dim
    assert scales.shape == (rows, dim // size)
    cut = ref.view(rows, -1, size)
    most = 448 if out == torch.float8_e4m3fn else 127
    want = cut.abs().amax(-1) / most
    want = torch.where(want > 0, want, 1.0)
    err = (GROWTH + 2) * 2.0 ** -24
    assert ((scales.double() - want).abs() <= err * want).all()
    assert (scales[-1] == 1).all() and not q[-1].float().any()
    s = scales.double().unsqueeze(-1)
    got = q.double().view(cut.shape) * s
    half = 0.5 * s if out == torch.int8 else 2.0 ** -4 * cut.abs() + 2.0 ** -10 * s
    assert ((got - cut).abs() <= half + 2 * err * (cut.abs() + s)).all()
    # without a residual: of the sum, the same bits
    again = F.rms_norm_quantized(total.to(dtype), w, None, EPS, group, out)
    assert len(again) == 2
    if stream == dtype:
        assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(again[1], scales)


def test_quantized_feeds_an_8_bit_product():
    """The scaled product of 8-bit rows and weights that the values are made for, against the
    product of the values they stand for: bf16 out rounds once, sums are 32 bits."""
    x, r, w = _case(64, 256, BF16)
    q, scales, _ = F.rms_norm_quantized(x, w, r)
    other = torch.randn(128, 256, device=DEV)
    side = other.abs().amax(1, keepdim=True) / 448
    p = (other / side).to(torch.float8_e4m3fn)
    got = torch._scaled_mm(q, p.t(), scale_a=scales, scale_b=side.t().contiguous(),
                           out_dtype=BF16)
    a, b = q.double() * scales.double(), p.double() * side.double()
    ref, spread = a @ b.t(), a.abs() @ b.abs().t()
    assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -12 * spread).all()


def test_infinities_and_nan_stay_in_their_rows():
    for out in (None, torch.float8_e4m3fn, torch.int8):
        x, r, w = _case(5, 256, BF16)
        x[1, 3], x[3, 7] = float("inf"), float("nan")
        if out is None:
            y = F.rms_norm(x, w, r)[0].float()
            assert torch.isnan(y[3]).all() and torch.isnan(y[1, 3])
        else:
            q, scales, _ = F.rms_norm_quantized(x, w, r, dtype=out, group_size=128)
            y = q.float() * scales.repeat_interleave(128, 1)
            assert torch.isnan(scales[3]).all() and torch.isnan(scales[1, 0])
        assert torch.isfinite(y[[0, 2, 4]]).all()


def test_empty_and_strided():
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.empty(0, 8, device=DEV, requires_grad=True)
    y, total = F.rms_norm(x, w, torch.empty(0, 8, device=DEV))
    assert y.shape == total.shape == (0, 8)
    assert not torch.autograd.grad(y.sum(), w)[0].any()
    assert F.rms_norm_quantized(x.detach(), w.detach(), group_size=4)[1].shape == (0, 2)
    x = torch.randn(6, 4, 8, device=DEV).transpose(0, 1)
    assert torch.equal(F.rms_norm(x, None), F.rms_norm(x.contiguous(), None))
    assert F.RMSNorm(8).to(DEV)(x).shape == x.shape


def test_another_stream_and_a_graph():
    x, r, w = _case(300, 1000, BF16)
    want = F.rms_norm(x, w, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.rms_norm(x, w, r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for t in (x, r, w):
        t.requires_grad_()
    dy = torch.randn_like(want[0])

    def step():
        y, total = F.rms_norm(x, w, r)
        return (y.detach(), total.detach(), *torch.autograd.grad((y, total), (x, r, w), (dy, dy)))

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_refusals():
    x, r, w = _case(4, 16, BF16)
    with pytest.raises(ValueError, match="residual"):
        F.rms_norm(x, w, r[:2])
    with pytest.raises(TypeError, match="residual"):
        F.rms_norm(x, w, r.half())
    with pytest.raises(TypeError, match="weight"):
        F.rms_norm(x, w.half())
    with pytest.raises(ValueError, match="weight"):
        F.rms_norm(x, w[:3])
    with pytest.raises(ValueError, match="eps"):
        F.rms_norm(x, w, eps=-1.0)
    with pytest.raises(TypeError):
        F.rms_norm(x.int())
    with pytest.raises(RuntimeError, match="CUDA"):
        F.rms_norm(x, w, r.cpu())
    with pytest.raises(ValueError, match="divide"):
        F.rms_norm_quantized(x, w, group_size=5)
    with pytest.raises(ValueError, match="divide"):
        F.rms_norm_quantized(x, w, group_size=0)
    with pytest.raises(TypeError, match="dtype"):
        F.rms_norm_quantized(x, w, dtype=torch.uint8)
    with pytest.raises(TypeError, match="float64"):
        F.rms_norm_quantized(x.double())
    with pytest.raises(RuntimeError, match="no gradient"):
        F.rms_norm_quantized(x.float().requires_grad_())
    y, _ = F.rms_norm(x.float().requires_grad_(), residual=r.float())
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable,
                                create_graph=True)[0]
        g.sum().backward()
