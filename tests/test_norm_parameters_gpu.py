"""layer_norm with parameters that begin anywhere: fp32 weights and biases beside 16-bit rows, and
views into a flat buffer, whose first element is on no boundary but its own.  The tolerances are
those of test_norm_gpu."""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from .test_norm_gpu import DEV, _case, _check, _reference

pytestmark = pytest.mark.gpu


def _at(t, offset):
    """``t``'s values in a view ``offset`` elements into a buffer of its own."""
    flat = torch.empty(t.numel() + offset, device=t.device, dtype=t.dtype)
    flat[offset:] = t.flatten()
    return flat[offset:].view(t.shape)


@pytest.mark.parametrize("dtype,param", [
    (torch.float16, torch.float32), (torch.bfloat16, torch.float32),
    (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
    (torch.float32, torch.float32), (torch.float64, torch.float64)])
@pytest.mark.parametrize("rows,dim", [(5, 2), (3, 31), (7, 130), (9, 256), (11, 384), (13, 1001),
                                      (13, 1002), (2, 4096), (2, 12290)])
@pytest.mark.parametrize("offset", [0, 1, 2, 3])
def test_parameters_at_any_offset(rows, dim, dtype, param, offset):
    x, w, b, dy = _case(rows, dim, dtype, param, seed=dim)
    # the weight and the bias at offsets of their own, and rows that do or do not start with them
    weight, bias = _at(w, offset), _at(b, (offset + 2) % 4)
    eps = 1e-3 if dim < 4 else 1e-5
    for rows_at in (x, _at(x, 2)):
        leaves = [t.requires_grad_() for t in (rows_at, weight, bias)]
        y = F.layer_norm(*leaves, eps)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        assert dw.dtype == db.dtype == param
        with torch.no_grad():
            ry, shift, rdx, rdw, rdb, rstd, h, g = _reference(x, w, b, eps, dy)
            wmax = w.double().abs().amax()
            _check(y, ry, dtype, (1 + shift + h.abs()) * wmax + b.double().abs(), "y")
            gmax = g.abs().amax(-1, keepdim=True)
            hmax = 1 + h.abs().amax(-1, keepdim=True)
            _check(dx, rdx, dtype, rstd * gmax * hmax * (hmax + shift), "dx")
            _check(dw, rdw, param, (dy.double().abs() * (h.abs() + shift + 1)).sum(0), "dweight")
            _check(db, rdb, param, dy.double().abs().sum(0), "dbias")
        only = F.layer_norm(rows_at.detach(), weight.detach(), None, eps)  # a weight alone
        _check(only, ry - b.double(), dtype, (1 + shift + h.abs()) * wmax, "y without bias")
