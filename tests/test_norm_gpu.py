"""layer_norm and its gradients against the formula in 64 bits.

Tolerances, set from the arithmetic: a result rounded once to a type of unit roundoff u is off by
u |result|; the sums run in 32 bits over trees and short runs, so a row's mean and sum of squares
are off by at most about (log2 D + 16) 2^-24 of the sum of magnitudes, written here as
``GROWTH`` = 48 roundings, times the largest magnitude that enters.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROUND = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
         torch.bfloat16: 2.0 ** -8}
ACC = {torch.float64: 2.0 ** -53}
GROWTH = 48
TINY = {torch.float64: 0.0, torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}


def _reference(x, w, b, eps, dy=None):
    x = x.double()
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(x[0]) if b is None else b.double()
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(centred.square().mean(-1, keepdim=True) + eps)
    h = centred * rstd
    y = h * w + b
    # rounding of the mean moves every centred value by this much
    shift = (x.abs().amax(-1, keepdim=True) * rstd)
    if dy is None:
        return y, shift
    dy = dy.double()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return y, shift, dx, (dy * h).sum(0), dy.sum(0), rstd, h, g


def _check(got, ref, dtype, spread, what):
    bound = (ROUND[dtype] * ref.abs() + GROWTH * ACC.get(dtype, 2.0 ** -24) * spread
             + TINY[dtype])
    worst = ((got.double() - ref).abs() / bound.clamp(min=1e-300)).max()
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


def _case(rows, dim, dtype, param, seed=0, offset=3.0):
    torch.manual_seed(seed)
    x = (torch.randn(rows, dim, device=DEV) * 2 + offset).to(dtype)
    w = (1 + 0.2 * torch.randn(dim, device=DEV)).to(param)
    b = torch.randn(dim, device=DEV).to(param)
    dy = torch.randn(rows, dim, device=DEV).to(dtype)
    return x, w, b, dy


SHAPES = [(1, 1), (3, 2), (5, 31), (4, 32), (2, 100), (7, 255), (9, 256), (300, 257), (65, 1000),
          (33, 1001), (4, 2048), (3, 4097), (2, 8192), (2, 10001), (2, 16384), (1, 40001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_forward_and_gradients(rows, dim, dtype):
    x, w, b, dy = _case(rows, dim, dtype, dtype)
    for t in (x, w, b):
        t.requires_grad_()
    eps = 1e-3 if dim < 4 else 1e-5
    y = F.layer_norm(x, w, b, eps)
    assert y.dtype == dtype and y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        ry, shift, rdx, rdw, rdb, rstd, h, g = _reference(x, w, b, eps, dy)
        wmax = w.double().abs().amax()
        _check(y, ry, dtype, (1 + shift + h.abs()) * wmax + b.double().abs(), "y")
        gmax = g.abs().amax(-1, keepdim=True)
        hmax = 1 + h.abs().amax(-1, keepdim=True)
        # h is off by `shift` roundings (the mean) wherever it appears
        _check(dx, rdx, dtype, rstd * gmax * hmax * (hmax + shift), "dx")
        _check(dw, rdw, dtype, (dy.double().abs() * (h.abs() + shift + 1)).sum(0), "dweight")
        _check(db, rdb, dtype, dy.double().abs().sum(0), "dbias")
    with torch.no_grad():  # the path without statistics gives the same bits
        assert torch.equal(F.layer_norm(x, w, b, eps), y)


# rows that start anywhere, around the lengths at which the threads or the groups a thread change
ODD = [(11, d) for d in (127, 129, 191, 193, 383, 385, 511, 513, 767, 769, 1023, 1025, 1535, 1537,
                         2047, 2049, 2999, 4095)]
PAIRS = [(9, d) for d in (258, 382, 386, 514, 770, 1022, 1026, 1538, 2050, 6146, 8190, 8194)]
MANY = [(20000, 193), (3000, 491), (3001, 490)]  # the backward pass's blocks take several rows each


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", ODD + PAIRS + MANY)
def test_rows_of_single_elements_and_pairs(rows, dim, dtype):
    x, w, b, dy = _case(rows, dim, dtype, dtype, seed=dim)
    ry, shift = _reference(x, w, b, 1e-5)
    spread = (1 + shift + ry.abs()) * w.double().abs().amax() + 2 * b.double().abs().amax()
    _check(F.layer_norm(x, w, b), ry, dtype, spread, "y")
    plain, shift = _reference(x, None, None, 1e-5)
    _check(F.layer_norm(x), plain, dtype, 1 + shift + plain.abs(), "y without parameters")
    for t in (x, w, b):
        t.requires_grad_()
    dx, dw, db = torch.autograd.grad(F.layer_norm(x, w, b), (x, w, b), dy)
    with torch.no_grad():
        _, shift, rdx, rdw, rdb, rstd, h, g = _reference(x, w, b, 1e-5, dy)
        gmax = g.abs().amax(-1, keepdim=True)
        hmax = 1 + h.abs().amax(-1, keepdim=True)
        _check(dx, rdx, dtype, rstd * gmax * hmax * (hmax + shift), "dx")
        _check(dw, rdw, dtype, (dy.double().abs() * (h.abs() + shift + 1)).sum(0), "dweight")
        _check(db, rdb, dtype, dy.double().abs().sum(0), "dbias")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fp32_parameters_and_partial_needs(dtype):
    x, w, b, dy = _case(50, 384, dtype, torch.float32)
    w.requires_grad_()
    y = F.layer_norm(x, w, None)
    (dw,) = torch.autograd.grad(y, w, dy)
    ref = _reference(x, w.detach(), None, 1e-5, dy)
    assert dw.dtype == torch.float32
    _check(dw, ref[3], torch.float32, (dy.double().abs() * (ref[6].abs() + ref[1] + 1)).sum(0),
           "dweight")
    x.requires_grad_()
    (dx,) = torch.autograd.grad(F.layer_norm(x), x, dy)
    ref = _reference(x.detach(), None, None, 1e-5, dy)
    hmax = 1 + ref[6].abs().amax(-1, keepdim=True)
    _check(dx, ref[2], dtype, ref[5] * ref[7].abs().amax(-1, keepdim=True) * hmax
           * (hmax + ref[1]), "dx without parameters")


def test_large_mean_keeps_the_variance():
    """A mean 1000 times the spread: mean square minus squared mean would lose it."""
    torch.manual_seed(1)
    x = torch.randn(64, 768, device=DEV) + 1000.0
    y = F.layer_norm(x)
    ref, shift = _reference(x, None, None, 1e-5)[:2]
    _check(y, ref, torch.float32, 1 + shift + ref.abs(), "y")


def test_many_rows_and_repeatability():
    x, w, b, dy = _case(20011, 72, torch.float32, torch.float32)
    for t in (x, w, b):
        t.requires_grad_()
    first = torch.autograd.grad(F.layer_norm(x, w, b), (x, w, b), dy)
    again = torch.autograd.grad(F.layer_norm(x, w, b), (x, w, b), dy)
    for p, r in zip(first, again):
        assert torch.equal(p, r)
    with torch.no_grad():
        _, shift, _, rdw, rdb, _, h, _ = _reference(x, w, b, 1e-5, dy)
        _check(first[1], rdw, torch.float32, (dy.double().abs() * (h.abs() + shift + 1)).sum(0),
               "dweight")
        _check(first[2], rdb, torch.float32, dy.double().abs().sum(0), "dbias")


def test_gradients_by_differences():
    x, w, b, _ = _case(3, 9, torch.float64, torch.float64)
    for t in (x, w, b):
        t.requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: F.layer_norm(*a), (x, w, b))


def test_leading_axes_strides_and_misaligned_rows():
    torch.manual_seed(2)
    base = torch.randn(6, 5, 130, device=DEV)
    ref = _reference(base.reshape(-1, 130), None, None, 1e-5)[0].view(6, 5, 130)
    for x in (base, base.transpose(0, 1).contiguous().transpose(0, 1)):
        y = F.layer_norm(x)
        assert y.shape == x.shape
        assert (y.double() - ref).abs().max() <= 1e-5
    flat = torch.randn(1 + 4 * 256, device=DEV, dtype=torch.bfloat16)
    x = flat[1:].view(4, 256)  # rows that start 2 bytes past a 16-byte boundary
    assert torch.equal(F.layer_norm(x), F.layer_norm(x.clone()))


def test_non_finite_rows_stay_alone():
    x = torch.randn(9, 256, device=DEV)
    clean = F.layer_norm(x)
    x[4, 7] = float("inf")
    x[6, 0] = float("nan")
    y = F.layer_norm(x)
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(y[keep], clean[keep])
    assert y[6].isnan().all()


def test_empty_and_other_stream():
    w = torch.ones(16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    y = F.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w))
    side = torch.cuda.Stream()
    x = torch.randn(2000, 512, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = F.layer_norm(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, F.layer_norm(x))


def test_refusals():
    x = torch.randn(4, 16, device=DEV)
    with pytest.raises(ValueError, match="shape"):
        F.layer_norm(x, torch.ones(8, device=DEV))
    with pytest.raises(TypeError):
        F.layer_norm(x, torch.ones(16, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        F.layer_norm(x.double(), torch.ones(16, device=DEV))
    with pytest.raises(TypeError, match="one type"):
        F.layer_norm(x.half(), torch.ones(16, device=DEV), torch.ones(16, device=DEV).half())
    with pytest.raises(ValueError, match="eps"):
        F.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        F.layer_norm(torch.zeros(4, 0, device=DEV))
    with pytest.raises(TypeError):
        F.layer_norm(torch.zeros(4, 4, device=DEV, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        F.layer_norm(x, torch.ones(16))
    lib = _lib.load()
    assert lib.fdwt_layer_norm_forward(0, 0, 1, 0, x.data_ptr(), None, None, 1e-5, x.data_ptr(),
                                       None, None) == 1
    assert lib.fdwt_layer_norm_forward(0, 2, 1, 4, x.data_ptr(), None, None, 1e-5, x.data_ptr(),
                                       None, None) == 1
    assert lib.fdwt_layer_norm_backward(0, 0, 4, 16, x.data_ptr(), x.data_ptr(), None,
                                        x.data_ptr(), None, x.data_ptr(), None, None, 0, None) == 3
    with pytest.raises(RuntimeError):  # differentiable once
        x.requires_grad_()
        (g,) = torch.autograd.grad(F.layer_norm(x).square().sum(), x, create_graph=True)
        g.sum().backward()
