"""The norm, the short convolution and the scan where calls go wrong in use: what shared memory
held before, tensors of more than 2^31 elements, two streams at once, dual tensors, an update of a
state that a graph has saved.  Tolerances where values are compared: those of the operators' tests,
or the same bits."""

import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture
def filled():
    """Every kernel of the library after one that sets all shared memory to NaN."""
    def run(call):
        _lib.set_shared_memory_fill(True, 0xFFFFFFFF)
        try:
            result = call()
            torch.cuda.synchronize()
        finally:
            _lib.set_shared_memory_fill(False)
        return result
    return run


def _same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("dtype", [F32, BF16, F64])
@pytest.mark.parametrize("L,D,N,G", [(1, 8, 16, 1), (13, 66, 3, 3), (37, 130, 12, 1), (600, 70, 16, 1),
                                     (50, 24, 100, 2), (70, 33, 33, 1), (300, 260, 1, 1),
                                     (90, 64, 7, 2)])
def test_scan_reads_no_stale_shared_memory(L, D, N, G, dtype, filled):
    torch.manual_seed(L)
    wide = F64 if dtype == F64 else F32
    t = lambda *s, to=dtype: torch.randn(*s, device=DEV).to(to).requires_grad_()  # noqa: E731
    x, dt, gate, b, c = t(2, L, D), t(2, L, D), t(2, L, D), t(2, L, G, N), t(2, L, G, N)
    a = (-torch.rand(D, N, device=DEV)).to(wide).requires_grad_()
    skip, bias, first = t(D, to=wide), t(D, to=wide), t(2, D, N, to=wide)
    lengths = torch.tensor([L, max(0, L - 3)], device=DEV)
    inputs = (x, dt, a, b, c, skip, gate, bias, first)
    dy, df = torch.randn(2, L, D, device=DEV).to(dtype), torch.randn(2, D, N, device=DEV).to(wide)

    def call():
        y, f = F.selective_scan(x, dt, a, b, c, skip, gate, bias, True, first, lengths)
        return (y.detach(), f.detach(), *torch.autograd.grad((y, f), inputs, (dy, df)))

    def step():
        state = first.detach().clone()
        with torch.no_grad():
            y = F.selective_scan_step(x[:, 0], dt[:, 0], a, b[:, 0], c[:, 0], state, skip, gate[:, 0],
                                      bias, True)
        return y, state

    assert _same(filled(call), call())
    assert _same(filled(step), step())


@pytest.mark.parametrize("dtype", [F32, BF16, F64])
@pytest.mark.parametrize("L,D,W", [(1, 8, 2), (40, 33, 5), (333, 130, 4), (9, 1001, 8)])
def test_convolution_reads_no_stale_shared_memory(L, D, W, dtype, filled):
    torch.manual_seed(L)
    x, w, b, i = (torch.randn(*s, device=DEV).to(dtype).requires_grad_()
                  for s in ((2, L, D), (D, W), (D,), (2, W - 1, D)))
    lengths = torch.tensor([max(0, L - 2), L], device=DEV)
    dy = torch.randn(2, L, D, device=DEV).to(dtype)

    def call():
        y, f = F.causal_conv1d(x, w, b, "silu", i, lengths)
        return (y.detach(), f.detach(), *torch.autograd.grad(y, (x, w, b, i), dy))

    assert _same(filled(call), call())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,dim", [(3, 31), (9, 256), (7, 1001), (5, 2048), (2, 10001)])
def test_norm_reads_no_stale_shared_memory(rows, dim, dtype, filled):
    torch.manual_seed(dim)
    x, r, w = (torch.randn(*s, device=DEV).to(dtype).requires_grad_()
               for s in ((rows, dim), (rows, dim), (dim,)))
    d = torch.randn(rows, dim, device=DEV).to(dtype)

    def call():
        y, t = F.rms_norm(x, w, r)
        return (y.detach(), t.detach(), *torch.autograd.grad((y, t), (x, r, w), (d, d)))

    def quantized():
        with torch.no_grad():
            q, s, t = F.rms_norm_quantized(x, w, r, group_size=None if dim % 64 else 64)
        return q.view(torch.uint8), s, t

    assert _same(filled(call), call())
    assert _same(filled(quantized), quantized())


def test_more_than_2_to_31_elements():
    """Offsets past 32 bits: the end of a tensor of 2^31 and some elements against the same rows in a
    call of their own.  bf16 results of sums that differ in the last bits are a unit of 2^-8 apart at
    most, 2^-7 of the value; the values here are below 64."""
    L, D, tail = (1 << 20) + 40, 2048, 64
    assert L * D > 1 << 31
    w = torch.ones(D, device=DEV, dtype=BF16)
    x = torch.empty(1, L, D, device=DEV, dtype=BF16)
    x[:, :1000].normal_()
    x[:, 1000:-1000] = 0.25
    x[:, -1000:].normal_()
    with torch.no_grad():
        y, total = F.rms_norm(x, w, x)
        part = F.rms_norm(x[:, -tail:].contiguous(), w, x[:, -tail:].contiguous())
        assert torch.equal(y[:, -tail:], part[0]) and torch.equal(total[:, -tail:], part[1])
        del y, total
        taps = torch.randn(D, 4, device=DEV).to(BF16)
        y, last = F.causal_conv1d(x, taps)
        part, state = F.causal_conv1d(x[:, -tail:], taps, initial_state=x[:, -tail - 3:-tail].contiguous())
        assert torch.equal(y[:, -tail:], part) and torch.equal(last, state)
        del y
        a = -torch.rand(D, 4, device=DEV)
        bc = torch.randn(1, L, 1, 4, device=DEV).to(BF16)
        y, last = F.selective_scan(x, x, a, bc, bc, dt_softplus=True)
        cut = L - tail
        _, state = F.selective_scan(x[:, -1000:cut], x[:, -1000:cut], a, bc[:, -1000:cut],
                                    bc[:, -1000:cut], dt_softplus=True,
                                    initial_state=F.selective_scan(
                                        x[:, :-1000], x[:, :-1000], a, bc[:, :-1000],
                                        bc[:, :-1000], dt_softplus=True)[1])
        part, final = F.selective_scan(x[:, cut:], x[:, cut:], a, bc[:, cut:], bc[:, cut:],
                                       dt_softplus=True, initial_state=state)
        assert ((y[:, cut:] - part).abs().float() <= 2.0 ** -7 * part.abs().float() + 1e-3).all()
        assert ((last - final).abs() <= 1e-4 * final.abs() + 1e-4).all()


def test_two_streams_at_once():
    """Calls on two streams, each with workspaces of its own, give what they give alone."""
    torch.manual_seed(0)

    def case(seed):
        torch.manual_seed(seed)
        t = lambda *s: torch.randn(*s, device=DEV).to(BF16).requires_grad_()  # noqa: E731
        x, dt, b, c = t(1, 2000, 128), t(1, 2000, 128), t(1, 2000, 1, 16), t(1, 2000, 1, 16)
        a = (-torch.rand(128, 16, device=DEV)).requires_grad_()
        dy = torch.randn(1, 2000, 128, device=DEV).to(BF16)

        def call():
            y, f = F.selective_scan(x, dt, a, b, c, dt_softplus=True)
            return (y.detach(), f.detach(), *torch.autograd.grad(y, (x, dt, a, b, c), dy))
        return call

    calls = [case(1), case(2)]
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for k, (s, call) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[k].append(call())
    torch.cuda.synchronize()
    for k in range(2):
        assert all(_same(g, want[k]) for g in got[k])


def test_dual_tensors_raise():
    x = torch.randn(2, 5, 8, device=DEV)
    w, a = torch.randn(8, 3, device=DEV), -torch.rand(8, 4, device=DEV)
    bc = torch.randn(2, 5, 1, 4, device=DEV)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: F.rms_norm(d), lambda: F.rms_norm(x, residual=d),
                     lambda: F.rms_norm_quantized(d), lambda: F.causal_conv1d(d, w),
                     lambda: F.selective_scan(d, x, a, bc, bc),
                     lambda: F.causal_conv1d_step(d[:, 0], w, torch.zeros(2, 2, 8, device=DEV)),
                     lambda: F.selective_scan_step(d[:, 0], x[:, 0], a, bc[:, 0], bc[:, 0],
                                                   torch.zeros(2, 8, 4, device=DEV))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()


def test_second_derivatives_raise():
    x = torch.randn(2, 5, 8, device=DEV, requires_grad=True)
    w, a = torch.randn(8, 3, device=DEV), -torch.rand(8, 4, device=DEV)
    bc = torch.randn(2, 5, 1, 4, device=DEV)
    for call in (lambda: F.rms_norm(x), lambda: F.causal_conv1d(x, w)[0],
                 lambda: F.selective_scan(x, x, a, bc, bc)[0]):
        g, = torch.autograd.grad(call().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|twice"):
            g.sum().backward()


def test_shared_and_broadcast_inputs():
    """One tensor as x, dt and gate, b and c expanded over tokens: gradients add up."""
    torch.manual_seed(4)
    x = torch.randn(2, 30, 24, device=DEV, dtype=F64, requires_grad=True)
    row = torch.randn(2, 1, 1, 5, device=DEV, dtype=F64, requires_grad=True)
    a = -torch.rand(24, 5, device=DEV, dtype=F64)
    b = row.expand(2, 30, 1, 5)
    y, _ = F.selective_scan(x, x, a, b, b, gate=x, dt_softplus=True)
    y.square().sum().backward()
    xs = [x.detach().clone().requires_grad_() for _ in range(3)]
    bs = [b.detach().clone().requires_grad_() for _ in range(2)]
    z, _ = F.selective_scan(xs[0], xs[1], a, bs[0], bs[1], gate=xs[2], dt_softplus=True)
    z.square().sum().backward()
    assert torch.allclose(y, z, rtol=1e-13, atol=1e-13)
    assert torch.allclose(x.grad, sum(t.grad for t in xs), rtol=1e-11, atol=1e-11)
    assert torch.allclose(row.grad, sum(t.grad for t in bs).sum(1, keepdim=True), rtol=1e-11, atol=1e-11)


FIRST_CALLS = """
import torch
import pytorch_morlet_fdwt_b200 as F
t = lambda *s: torch.randn(*s, device="cuda").bfloat16().requires_grad_()
x, w, g, bc, dy = t(2, 300, 64), t(64, 4), t(64), t(2, 300, 1, 16), t(2, 300, 64).detach()
a = (-torch.rand(64, 16, device="cuda")).requires_grad_()
states, inputs = torch.zeros(2, 64, 16, device="cuda"), torch.zeros(2, 3, 64, device="cuda").bfloat16()

def run():
    out = [*torch.autograd.grad(F.rms_norm(x, g, x)[0], (x, g), dy),
           *torch.autograd.grad(F.causal_conv1d(x, w, None, "silu")[0], (x, w), dy),
           *torch.autograd.grad(F.selective_scan(x, x, a, bc, bc, dt_softplus=True)[0], (x, a, bc), dy)]
    with torch.no_grad():
        out += F.rms_norm_quantized(x, g, group_size=32)
        out.append(F.causal_conv1d_step(x[:, 0], w, inputs))
        out.append(F.selective_scan_step(x[:, 0], x[:, 0], a, bc[:, 0], bc[:, 0], states,
                                         dt_softplus=True))
    return out

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = run()
graph.replay()
torch.cuda.synchronize()
states.zero_(), inputs.zero_()
want = run()
assert all(torch.equal(p.float(), q.float()) for p, q in zip(held, want))
"""


def test_first_calls_in_a_capture():
    """A process whose first call of every operator is captured in a graph."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", FIRST_CALLS], check=True, cwd=root, timeout=300)
