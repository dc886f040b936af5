"""SelectiveTokenMixer and SelectiveTokenStack: training, prompts, single tokens, against the same
layer written out in 64 bits.

In fp32 (whose matrix products torch runs in 32 bits) a layer's values come from some thousand
roundings of magnitudes near one: 2^-24 times 1000 is 6e-5 relative to the largest value, taken
as 1e-4, for gradients relative to each one's largest.  bf16 rounds after each of about ten steps,
2^-8 each with random signs along rows of 64 to 128 terms: 5 % of the largest value.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _norm(x, w, eps=1e-6):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _reference(P, x, lengths=None, prefix=""):
    """The layer's mix of (B, L, D) tokens in fp64, token by token, without the residual."""
    g = lambda k: P[prefix + k]  # noqa: E731
    B, L, _ = x.shape
    E, W = g("conv_weight").shape
    N = g("log_rate").shape[1]
    h = _norm(x, g("norm.weight"))
    u, gate = (h @ g("in_proj.weight").T).split(E, -1)
    pad = torch.cat([u.new_zeros(B, W - 1, E), u], 1)
    p = sum(g("conv_weight")[:, j] * pad[:, j:j + L] for j in range(W)) + g("conv_bias")
    u = p * torch.sigmoid(p)
    low, b, c = (u @ g("x_proj.weight").T).split((g("dt_proj.weight").shape[1], N, N), -1)
    delta = torch.nn.functional.softplus(low @ g("dt_proj.weight").T + g("dt_bias"), threshold=50)
    rates = -torch.exp(g("log_rate"))
    state, out = x.new_zeros(B, E, N), []
    for t in range(L):
        state = (torch.exp(delta[:, t].unsqueeze(-1) * rates) * state
                 + (delta[:, t] * u[:, t]).unsqueeze(-1) * b[:, t].unsqueeze(1))
        out.append((state * c[:, t].unsqueeze(1)).sum(-1) + g("skip") * u[:, t])
    y = torch.stack(out, 1) * gate * torch.sigmoid(gate)
    return y @ g("out_proj.weight").T


def _params(module):
    return {k: p.detach().double().requires_grad_() for k, p in module.named_parameters()}


def _near(got, ref, tol, what):
    err = float((got.detach().double() - ref.detach()).abs().max())
    assert err <= tol * max(float(ref.detach().abs().max()), 1e-30), f"{what}: {err}"


@pytest.mark.parametrize("dim,L,options", [
    (32, 40, {}), (24, 150, {"state_size": 5, "conv_size": 3, "expand": 3, "dt_rank": 4}),
    (64, 9, {"state_size": 33})])
def test_layer_and_gradients(dim, L, options):
    torch.manual_seed(dim)
    layer = F.SelectiveTokenMixer(dim, **options).to(DEV)
    x = torch.randn(2, L, dim, device=DEV, requires_grad=True)
    y = layer(x)
    dy = torch.randn_like(y)
    y.backward(dy)
    P = _params(layer)
    xo = x.detach().double().requires_grad_()
    yo = xo + _reference(P, xo)
    yo.backward(dy.double())
    _near(y, yo, 1e-4, "y")
    _near(x.grad, xo.grad, 1e-4, "dL/dx")
    for k, p in layer.named_parameters():
        _near(p.grad, P[k].grad, 1e-4, f"dL/d{k}")


def test_prompts_and_single_tokens():
    torch.manual_seed(1)
    layer = F.SelectiveTokenMixer(48).to(DEV)
    x = torch.randn(3, 60, 48, device=DEV)
    lengths = torch.tensor([50, 0, 7], device=DEV)
    want = x.double() + _reference(_params(layer), x.double())
    with torch.no_grad():
        y, state = layer(x, lengths=lengths, return_state=True)
        for i, n in enumerate(lengths.tolist()):
            _near(y[i, :n], want[i, :n], 1e-4, "prompt") if n else None
        # pools: sequence i's state in slot 4 - i
        pools = layer.init_state(6, DEV)
        slots = torch.tensor([4, 3, 2], device=DEV)
        for pool, s in zip(pools, state):
            pool[slots] = s
        for k in range(6):
            at = lengths + k
            token = x[torch.arange(3), at]
            out = layer.step(token, pools, slots=slots)
            _near(out, want[torch.arange(3), at], 1e-4, f"token {k}")
        assert not any(p[[0, 1, 5]].any() for p in pools)
        # a prompt in two parts
        first, state = layer(x[:, :33], return_state=True)
        rest = layer(x[:, 33:], state=state)
        _near(torch.cat([first, rest], 1), want, 1e-4, "two parts")


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 0.05)])
def test_stack(dtype, tol):
    torch.manual_seed(2)
    stack = F.SelectiveTokenStack(32, 3, state_size=8).to(DEV).to(dtype)
    x = torch.randn(2, 30, 32, device=DEV).to(dtype).requires_grad_()
    y, states = stack(x, return_state=True)
    P = _params(stack)
    xo = x.detach().double().requires_grad_()
    total = xo
    for i in range(3):
        total = total + _reference(P, total, prefix=f"layers.{i}.")
    yo = _norm(total, P["norm.weight"])
    _near(y, yo, tol, "y")
    dy = torch.randn_like(y)
    y.backward(dy)
    if dtype == torch.float32:
        yo.backward(dy.double())
        _near(x.grad, xo.grad, tol, "dL/dx")
        for k, p in stack.named_parameters():
            _near(p.grad, P[k].grad, tol, f"dL/d{k}")
    else:
        assert all(torch.isfinite(p.grad).all() for p in stack.parameters())
    assert len(states) == 3
    # single tokens carry the whole stack's states on
    with torch.no_grad():
        _, states = stack(x[:, :20].detach(), return_state=True)
        for t in range(20, 30):
            out = stack.step(x[:, t].detach(), states)
        _near(out, yo[:, 29], tol, "single tokens")


def test_a_captured_token():
    """A token of the stack captured in a graph and replayed gives what the calls give."""
    torch.manual_seed(3)
    stack = F.SelectiveTokenStack(64, 2).to(DEV).to(torch.bfloat16)
    states, others = (stack.init_state(4, DEV, torch.bfloat16) for _ in range(2))
    x = torch.randn(4, 64, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        stack.step(x, stack.init_state(4, DEV, torch.bfloat16))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = stack.step(x, states)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        assert torch.equal(stack.step(x, others), held)
    for a, b in zip(states, others):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals():
    layer = F.SelectiveTokenMixer(16).to(DEV)
    stack = F.SelectiveTokenStack(16, 2).to(DEV)
    x = torch.randn(2, 5, 16, device=DEV)
    for module in (layer, stack):
        with pytest.raises(ValueError, match="B, L, D"):
            module(x[0])
        with pytest.raises(ValueError, match="B, D"):
            module.step(x, module.init_state(2, DEV))
    with pytest.raises(ValueError, match="2 states"):
        stack(x, state=stack.init_state(2, DEV)[:1])
    with pytest.raises(ValueError, match="depth"):
        F.SelectiveTokenStack(16, 0)
