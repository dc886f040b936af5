"""Layer norm and linear attention without a GPU: refusals, the C ABI's argument checks, its
descriptor's layout and workspace sizes."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib
from pytorch_morlet_fdwt_b200.linear_attention import _Desc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3


def _desc(dtype=3, heads=4, kv_heads=2, dk=64, dv=64, batch=2, length=1000):
    d = _Desc(dtype, heads, kv_heads, dk, dv, batch, length)
    d.q_stride[:] = (length * heads * dk, heads * dk, dk)
    d.k_stride[:] = (length * kv_heads * dk, kv_heads * dk, dk)
    d.v_stride[:] = (length * kv_heads * dv, kv_heads * dv, dv)
    d.o_stride[:] = (length * heads * dv, heads * dv, dv)
    d.scale = 1.0
    return d


def test_cpu_tensors_are_refused():
    x = torch.randn(2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.layer_norm(x)
    q = torch.randn(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        F.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        F.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))


def test_descriptor_layout_matches_the_header(tmp_path):
    """The ctypes mirror has the header's size and offsets, as a C compiler lays them out."""
    fields = [f[0] for f in _Desc._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fdwt_b200.h"\nint main(void) {\n'
                   '  printf("%zu", sizeof(fdwt_linattn_desc));\n'
                   + "".join(f'  printf(" %zu", offsetof(fdwt_linattn_desc, {f}));\n' for f in fields)
                   + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(n) for n in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(_Desc)] + [getattr(_Desc, f).offset for f in fields]


def test_c_entries_check_their_arguments():
    lib = _lib.load()
    ok = 4096  # a pointer that no call below reaches
    for bad in (_desc(dtype=9), _desc(heads=3), _desc(kv_heads=0), _desc(dk=0), _desc(dv=-1),
                _desc(batch=-1), _desc(length=-2)):
        at = ctypes.addressof(bad)
        assert lib.fdwt_linattn_forward(at, *[ok] * 9, 1 << 40, None) == INVALID
        assert lib.fdwt_linattn_backward(at, *[ok] * 13, 1 << 40, None) == INVALID
        assert lib.fdwt_linattn_step(at, *[ok] * 5, 8, None, ok, None) == INVALID
        assert lib.fdwt_linattn_forward_workspace(at) == 0
    wide = ctypes.addressof(d := _desc(dk=257))
    assert lib.fdwt_linattn_forward(wide, *[ok] * 9, 1 << 40, None) == UNSUPPORTED
    good = ctypes.addressof(e := _desc())
    assert lib.fdwt_linattn_forward(good, None, *[ok] * 8, 1 << 40, None) == INVALID
    assert lib.fdwt_linattn_step(good, *[ok] * 5, 8, None, ok, None) == INVALID  # length is not 1
    one = ctypes.addressof(f := _desc(length=1))
    assert lib.fdwt_linattn_step(one, *[ok] * 5, 1, None, ok, None) == INVALID  # too few states
    need = lib.fdwt_linattn_backward_workspace(good)
    assert need > 0 and lib.fdwt_linattn_backward(good, *[ok] * 12, None, 0, None) == WORKSPACE
    assert lib.fdwt_linattn_backward(good, *[ok] * 13, need - 1, None) == WORKSPACE
    empty = ctypes.addressof(g := _desc(batch=0))
    assert lib.fdwt_linattn_forward(empty, *[None] * 9, 0, None) == OK
    assert lib.fdwt_layer_norm_forward(0, 0, 0, 8, None, None, None, 1e-5, None, None, None) == OK
    assert lib.fdwt_layer_norm_forward(0, 0, 1, 8, None, None, None, 1e-5, ok, None, None) == INVALID
    assert lib.fdwt_layer_norm_forward(0, 1, 1, 8, ok, ok, None, 1e-5, ok, None, None) == INVALID
    assert lib.fdwt_layer_norm_forward(0, 0, 1, 8, ok, None, None, -1.0, ok, None, None) == INVALID
    assert lib.fdwt_layer_norm_backward(0, 0, 4, 8, ok, ok, None, ok, ok, ok, ok, None, 0,
                                        None) == WORKSPACE
    del d, e, f, g


def test_workspace_sizes():
    lib = _lib.load()
    # one block a head: nothing to hand over; few heads and a long sequence: states of segments
    many, few = _desc(heads=64, kv_heads=64, batch=8), _desc(heads=1, kv_heads=1, batch=1, length=1 << 20)
    assert lib.fdwt_linattn_forward_workspace(ctypes.addressof(many)) == 0
    assert lib.fdwt_linattn_forward_workspace(ctypes.addressof(few)) >= 64 * 64 * 4
    # shared heads: every query head's own gradients of k and v in 32 bits
    shared = _desc(heads=4, kv_heads=1)
    assert lib.fdwt_linattn_backward_workspace(ctypes.addressof(shared)) >= 2 * 1000 * 4 * 128 * 4
    assert lib.fdwt_layer_norm_backward_workspace(0, 100, 64, 0) == 0
    assert lib.fdwt_layer_norm_backward_workspace(0, 100, 64, 1) >= 2 * 64 * 4


def test_layers_construct_on_the_cpu():
    torch.manual_seed(0)
    layer = F.DecayTokenMixer(24, num_heads=4, num_kv_heads=2, head_dim=8, value_dim=6)
    assert layer.qkv_proj.out_features == 4 * 8 + 2 * (8 + 6)
    assert layer.out_proj.in_features == 4 * 6
    a = layer.log_decay("cpu")
    assert a.dtype == torch.float32 and (a < 0).all() and (a[1:] > a[:-1]).all()
    assert layer.to(torch.bfloat16).log_decay("cpu").dtype == torch.float32
    assert layer.init_state(3, "cpu").shape == (3, 4, 8, 6)
    assert set(F.LayerNorm(5).state_dict()) == {"weight", "bias"}


def test_package_exports():
    code = ("import pytorch_morlet_fdwt_b200 as F; "
            "assert callable(F.linear_attention) and callable(F.layer_norm); "
            "assert all(hasattr(F, n) for n in F.__all__)")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)
