"""The selective mixer's operators without a GPU: refusals, the C ABI's argument checks, its
descriptors' layout and workspace sizes, the layers' parameters."""

import ctypes
import os
import subprocess

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib
from pytorch_morlet_fdwt_b200.causal_conv import _ConvDesc
from pytorch_morlet_fdwt_b200.selective_scan import _ScanDesc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
PTR = 4096  # a pointer that no call below reaches


def _conv(dtype=3, param=3, width=4, batch=2, length=100, dim=64):
    d = _ConvDesc(dtype, param, width, 1, batch, length, dim)
    d.x_stride[:] = d.dy_stride[:] = (length * dim, dim)
    return d


def _scan(dtype=3, groups=1, states=16, batch=2, length=100, dim=64):
    d = _ScanDesc(dtype, groups, states, 1, batch, length, dim)
    for s in (d.x_stride, d.dt_stride, d.gate_stride, d.dy_stride):
        s[:] = (length * dim, dim)
    d.b_stride[:] = d.c_stride[:] = (length * groups * states, groups * states, states)
    return d


def test_cpu_tensors_are_refused():
    x, w = torch.randn(2, 8, 16), torch.randn(16, 4)
    bc, a = torch.randn(2, 8, 1, 4), -torch.ones(16, 4)
    for call in (lambda: F.rms_norm(x), lambda: F.rms_norm(x, residual=x),
                 lambda: F.rms_norm_quantized(x), lambda: F.causal_conv1d(x, w),
                 lambda: F.causal_conv1d_step(x[:, 0], w, torch.zeros(2, 3, 16)),
                 lambda: F.selective_scan(x, x, a, bc, bc),
                 lambda: F.selective_scan_step(x[:, 0], x[:, 0], a, bc[:, 0], bc[:, 0],
                                               torch.zeros(2, 16, 4))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("mirror,name", [(_ConvDesc, "fdwt_conv1d_desc"),
                                         (_ScanDesc, "fdwt_scan_desc")])
def test_descriptor_layouts_match_the_header(mirror, name, tmp_path):
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fdwt_b200.h"\nint main(void) {\n'
                   f'  printf("%zu", sizeof({name}));\n'
                   + "".join(f'  printf(" %zu", offsetof({name}, {f}));\n' for f in fields)
                   + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(n) for n in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


def test_norm_entries_check_their_arguments():
    lib = _lib.load()
    fwd = lambda *c, x=PTR, r=None, y=PTR, t=None, eps=1e-6, rows=2, dim=8: (  # noqa: E731
        lib.fdwt_rms_norm_forward(*c, rows, dim, x, r, None, eps, y, t, None, None))
    for codes in ((9, 9, 9), (0, 1, 0), (3, 2, 3), (1, 0, 1), (3, 3, 1)):
        assert fwd(*codes) == INVALID
    assert fwd(0, 0, 0, rows=-1) == INVALID and fwd(0, 0, 0, dim=0) == INVALID
    assert fwd(0, 0, 0, eps=-1.0) == INVALID and fwd(0, 0, 0, x=None) == INVALID
    assert fwd(0, 0, 0, r=PTR) == INVALID and fwd(0, 0, 0, t=PTR) == INVALID
    assert fwd(0, 0, 0, rows=0, x=None, y=None) == OK
    quant = lambda kind, group, dtype=3, q=PTR, s=PTR, rows=2: lib.fdwt_rms_norm_quantized(  # noqa: E731
        dtype, dtype, dtype, kind, rows, 8, group, PTR, None, None, 1e-6, q, s, None, None)
    assert quant(2, 8) == INVALID and quant(0, 3) == INVALID and quant(0, 0) == INVALID
    assert quant(0, 8, q=None) == INVALID and quant(0, 8, s=None) == INVALID
    assert quant(0, 8, dtype=1) == UNSUPPORTED and quant(0, 8, rows=0) == OK
    need = lib.fdwt_rms_norm_backward_workspace(0, 100, 64, 1)
    assert need >= 64 * 4 and lib.fdwt_rms_norm_backward_workspace(0, 100, 64, 0) == 0
    back = lambda dx, dr, ws, n: lib.fdwt_rms_norm_backward(  # noqa: E731
        0, 0, 0, 100, 64, PTR, None, PTR, None, PTR, dx, dr, PTR, ws, n, None)
    assert back(PTR, None, None, 0) == WORKSPACE and back(PTR, None, PTR, need - 1) == WORKSPACE
    assert back(None, PTR, PTR, need) == INVALID


def test_convolution_entries_check_their_arguments():
    lib = _lib.load()
    for bad in (_conv(dtype=9), _conv(param=2), _conv(dtype=1, param=0), _conv(width=1),
                _conv(width=9), _conv(batch=-1), _conv(length=-1), _conv(dim=0)):
        at = ctypes.addressof(bad)
        assert lib.fdwt_causal_conv1d_forward(at, *[PTR] * 7, None) == INVALID
        assert lib.fdwt_causal_conv1d_backward(at, *[PTR] * 12, 1 << 40, None) == INVALID
        assert lib.fdwt_causal_conv1d_step(at, *[PTR] * 4, 8, None, PTR, None) == INVALID
        assert lib.fdwt_causal_conv1d_backward_workspace(at) == 0
    good = _conv()
    at = ctypes.addressof(good)
    assert lib.fdwt_causal_conv1d_forward(at, None, *[PTR] * 6, None) == INVALID
    assert lib.fdwt_causal_conv1d_step(at, *[PTR] * 4, 8, None, PTR, None) == INVALID  # length 100
    need = lib.fdwt_causal_conv1d_backward_workspace(at)
    assert need >= 5 * 64 * 4
    assert lib.fdwt_causal_conv1d_backward(at, *[PTR] * 12, need - 1, None) == WORKSPACE
    one = _conv(length=1)
    assert lib.fdwt_causal_conv1d_step(ctypes.addressof(one), *[PTR] * 4, 1, None, PTR,
                                       None) == INVALID  # too few states
    empty = _conv(batch=0)
    assert lib.fdwt_causal_conv1d_forward(ctypes.addressof(empty), *[None] * 8) == OK


def test_scan_entries_check_their_arguments():
    lib = _lib.load()
    for bad in (_scan(dtype=9), _scan(groups=0), _scan(groups=3), _scan(states=0), _scan(batch=-1),
                _scan(length=-1), _scan(dim=0)):
        at = ctypes.addressof(bad)
        assert lib.fdwt_selscan_forward(at, *[PTR] * 14, 1 << 40, None) == INVALID
        assert lib.fdwt_selscan_backward(at, *[PTR] * 22, 1 << 40, None) == INVALID
        assert lib.fdwt_selscan_step(at, *[PTR] * 9, 8, None, PTR, None) == INVALID
        assert lib.fdwt_selscan_forward_workspace(at) == 0
        assert lib.fdwt_selscan_checkpoint_bytes(at) == 0
    wide = _scan(states=129)
    at = ctypes.addressof(wide)
    assert lib.fdwt_selscan_forward(at, *[PTR] * 14, 1 << 40, None) == UNSUPPORTED
    assert lib.fdwt_selscan_backward(at, *[PTR] * 22, 1 << 40, None) == UNSUPPORTED
    good = _scan(batch=1, length=65536)
    at = ctypes.addressof(good)
    assert lib.fdwt_selscan_forward(at, None, *[PTR] * 13, 1 << 40, None) == INVALID
    need = lib.fdwt_selscan_forward_workspace(at)  # few channels: segments
    assert need > 0 and lib.fdwt_selscan_forward(at, *[PTR] * 14, need - 1, None) == WORKSPACE
    for off in (4, 16):  # off 32 bytes
        assert lib.fdwt_selscan_forward(at, *[PTR] * 13, PTR + off, need, None) == INVALID
    need = lib.fdwt_selscan_backward_workspace(at)
    assert lib.fdwt_selscan_backward(at, *[PTR] * 22, need - 1, None) == WORKSPACE
    # the states before every eighth token, padded to a power of two
    assert lib.fdwt_selscan_checkpoint_bytes(at) == 65536 // 8 * 64 * 16 * 4
    odd = _scan(states=9, length=17)
    assert lib.fdwt_selscan_checkpoint_bytes(ctypes.addressof(odd)) == 2 * 3 * 64 * 16 * 4
    one = _scan(length=1)
    assert lib.fdwt_selscan_step(ctypes.addressof(one), *[PTR] * 9, 1, None, PTR, None) == INVALID
    empty = _scan(batch=0)
    assert lib.fdwt_selscan_forward(ctypes.addressof(empty), *[None] * 14, 0, None) == OK


def test_layers_construct_on_the_cpu():
    torch.manual_seed(0)
    layer = F.SelectiveTokenMixer(24, state_size=6, conv_size=3, expand=3)
    assert layer.in_proj.out_features == 2 * 72 and layer.dt_rank == 2
    assert layer.conv_weight.shape == (72, 3) and layer.log_rate.shape == (72, 6)
    assert (layer._rates() < 0).all()
    size = torch.nn.functional.softplus(layer.dt_bias)
    assert (size > 9e-4).all() and (size < 0.11).all()
    conv, scan = layer.init_state(5, "cpu", torch.bfloat16)
    assert conv.shape == (5, 2, 72) and conv.dtype == torch.bfloat16
    assert scan.shape == (5, 72, 6) and scan.dtype == torch.float32
    stack = F.SelectiveTokenStack(16, 3)
    assert len(stack.layers) == 3 and len(stack.init_state(2, "cpu")) == 3
    assert set(F.RMSNorm(5).state_dict()) == {"weight"}
    assert all(hasattr(F, n) for n in F.__all__)
