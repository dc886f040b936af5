"""linear_attention, its gradients, linear_attention_step and DecayTokenMixer against the
definition in 64 bits.

Tolerances, set from the arithmetic: with A the same operator on absolute values, a sum of n
products in 32 bits is off by at most n 2^-24 A; n is taken as Dk + Dv + 128 + L/32 (a product
along a head, one along a chunk, and the chunks in turn).  16-bit types also round the scores, the
state's copy and the result (unit roundoff u): 2 u A + u |result| at worst, and 2 u of the root
mean square where the roundings are independent.  The state's update carries two 16-bit parts of
each value, u^2 (at most 2^-16) of A.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROUND = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11,
         torch.bfloat16: 2.0 ** -8}
HALF = (torch.float16, torch.bfloat16)


def _schedule(heads, fast=False):
    rate = torch.logspace(-1, 0.5, heads) if fast else torch.logspace(-3, -1, heads)
    return -rate.to(DEV)


def _inputs(B, L, H, Hk, Dk, Dv, dtype, seed=0, initial=False, lengths=None, fast=False):
    torch.manual_seed(seed)
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    q = torch.randn(B, L, H, Dk, device=DEV).to(dtype)
    k = torch.randn(B, L, Hk, Dk, device=DEV).to(dtype)
    v = torch.randn(B, L, Hk, Dv, device=DEV).to(dtype)
    s0 = torch.randn(B, H, Dk, Dv, device=DEV, dtype=acc) if initial else None
    n = None if lengths is None else torch.tensor(lengths, device=DEV)
    return q, k, v, _schedule(H, fast).to(acc), s0, n


def _reference(q, k, v, a, s0, n, scale):
    """The closed form over all pairs of tokens, in 64 bits (differentiable)."""
    q, k, v, a = q.double(), k.double(), v.double(), a.double()
    B, L, H, Dk = q.shape
    group = H // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    t = torch.arange(L, device=q.device)
    n = torch.full((B,), L, device=q.device) if n is None else n.clamp(0, L)
    live = (t < n.view(B, 1)).double().view(B, L, 1, 1)
    s0 = q.new_zeros(B, H, Dk, v.shape[-1]) if s0 is None else s0.double()
    gap = t.view(-1, 1) - t
    # 0 * -inf has no value: a power zero is one, and what the mask drops is zero
    power = a.view(H, 1, 1) * gap.clamp(min=1)
    mask = torch.where(gap == 0, 1.0, torch.where(gap > 0, power.exp(), 0.0))
    score = torch.einsum("blhd,bmhd->bhlm", q, k * live) * mask
    out = torch.einsum("bhlm,bmhe->blhe", score, v * live)
    read = (a.view(1, H) * (t + 1).view(L, 1)).exp()
    out = out + torch.einsum("blhd,bhde->blhe", q, s0) * read.view(1, L, H, 1)
    age = n.view(B, 1) - 1 - t
    weight = torch.where(age.unsqueeze(-1) == 0, 1.0,
                         (a.view(1, 1, H) * age.clamp(min=1).unsqueeze(-1)).exp()) * live[..., 0]
    final = torch.einsum("blhd,blhe->bhde", k * weight.unsqueeze(-1), v)
    whole = torch.where(n.view(B, 1) == 0, 1.0,
                        (a.view(1, H) * n.clamp(min=1).view(B, 1)).exp())
    return scale * out * live, final + whole.view(B, H, 1, 1) * s0


def _growth(L, Dk, Dv, dtype):
    unit = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    return (Dk + Dv + 128 + L / 32) * unit


def _check(got, ref, size, dtype, growth, what, state=False):
    """size: the operator on absolute values."""
    got, size = got.double(), size.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    half = dtype in HALF
    u = ROUND[dtype]
    bound = growth * size
    if half and state:
        bound = bound + 2.0 ** -16 * size
    elif half:
        bound = bound + 2 * u * size + u * ref.abs() + 2.0 ** -24
    worst = ((got - ref).abs() / (bound + 1e-300)).max() if ref.numel() else 0
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"
    if half and not state and ref.numel() > 1000:
        off = (got - ref).square().mean().sqrt()
        assert off <= 2 * u * ref.square().mean().sqrt(), f"{what}: rms {off:.3g}"


def _magnitudes(q, k, v, a, s0, n, scale):
    return _reference(q.abs(), k.abs(), v.abs(), a, None if s0 is None else s0.abs(), n, scale)


CASES = [  # B, L, H, Hkv, Dk, Dv, initial, lengths
    (1, 1, 1, 1, 1, 1, False, None),
    (2, 1, 2, 1, 16, 8, True, None),
    (1, 2, 3, 3, 5, 7, True, None),
    (2, 63, 2, 2, 64, 64, False, None),
    (1, 64, 4, 2, 64, 32, True, None),
    (3, 65, 2, 1, 32, 48, True, [65, 0, 1]),
    (1, 127, 2, 2, 128, 128, True, None),
    (2, 128, 2, 1, 64, 128, False, [128, 127]),
    (1, 129, 2, 2, 128, 64, True, None),
    (4, 300, 6, 2, 48, 80, True, [300, 129, 128, 0]),
    (2, 517, 2, 2, 33, 65, True, [300, 517]),
    (1, 640, 1, 1, 64, 64, True, None),
    (1, 700, 2, 1, 136, 200, True, None),
    (2, 385, 1, 1, 256, 256, False, None),
    (1, 1100, 1, 1, 128, 128, True, [1030]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,L,H,Hk,Dk,Dv,initial,lengths", CASES)
def test_forward_and_gradients(B, L, H, Hk, Dk, Dv, initial, lengths, dtype):
    q, k, v, a, s0, n = _inputs(B, L, H, Hk, Dk, Dv, dtype, L, initial, lengths)
    scale = Dk ** -0.5
    torch.manual_seed(L + 1)
    do = torch.randn(B, L, H, Dv, device=DEV).to(dtype)
    ds = torch.randn(B, H, Dk, Dv, device=DEV).to(a.dtype)
    wrt = [t.requires_grad_() for t in (q, k, v, s0) if t is not None]
    out, final = F.linear_attention(q, k, v, a, initial_state=s0, lengths=n)
    assert out.dtype == dtype and out.shape == (B, L, H, Dv) and final.dtype == a.dtype
    grads = torch.autograd.grad((out, final), wrt, (do, ds))
    rout, rfinal = _reference(q, k, v, a, s0, n, scale)
    rgrads = torch.autograd.grad((rout, rfinal), wrt, (do.double(), ds.double()))
    # the operator and its gradients are sums of products: on absolute values they bound the
    # rounding errors
    mags = [t.detach().abs().requires_grad_() for t in wrt]
    mout, mfinal = _reference(*mags[:3], a, mags[3] if initial else None, n, scale)
    mgrads = torch.autograd.grad((mout, mfinal), mags, (do.abs().double(), ds.abs().double()))
    growth = _growth(L, Dk, Dv, dtype)
    _check(out, rout, mout, dtype, growth, "out")
    _check(final, rfinal, mfinal, dtype, growth, "final state", state=True)
    # a sum over the heads that share a key adds a rounding a head
    for name, got, ref, mag in zip(("dq", "dk", "dv", "ds0"), grads, rgrads, mgrads):
        assert got.dtype == (a.dtype if name == "ds0" else dtype)
        extra = H // Hk if dtype in HALF and H != Hk and name in ("dk", "dv") else 0
        _check(got, ref, mag * (1 + extra), dtype, growth, name, state=name == "ds0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequence_in_segments(dtype):
    """Long enough to be cut into segments on every path; the reference runs in pieces."""
    B, L, H, D = 1, 9000, 2, 64
    q, k, v, a, s0, _ = _inputs(B, L, H, H, D, D, dtype, 3, True)
    out, final = F.linear_attention(q, k, v, a, initial_state=s0)
    state, mag, outs, mags = s0, s0.abs(), [], []
    for i in range(0, L, 500):
        part = [t[:, i:i + 500] for t in (q, k, v)]
        o, state = _reference(*part, a, state, None, D ** -0.5)
        m, mag = _magnitudes(*part, a, mag, None, D ** -0.5)
        outs.append(o)
        mags.append(m)
    growth = _growth(L, D, D, dtype)
    _check(out, torch.cat(outs, 1), torch.cat(mags, 1), dtype, growth, "out")
    _check(final, state, mag, dtype, growth, "final state", state=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_strong_and_total_decay(dtype):
    """Decays down to e^-3.2 a token, and one of zero (log decay -inf: only the token itself)."""
    q, k, v, a, s0, _ = _inputs(2, 200, 4, 4, 64, 64, dtype, 5, True, None, True)
    a[1] = -float("inf")
    a[2] = 0.0
    do = torch.randn(2, 200, 4, 64, device=DEV).to(dtype)
    wrt = [t.requires_grad_() for t in (q, k, v, s0)]
    out, final = F.linear_attention(q, k, v, a, initial_state=s0)
    grads = torch.autograd.grad((out, final), wrt, (do, torch.ones_like(final)))
    ref, rfinal = _reference(q, k, v, a, s0, None, 64 ** -0.5)
    rgrads = torch.autograd.grad((ref, rfinal), wrt, (do.double(), torch.ones_like(rfinal)))
    mags = [t.detach().abs().requires_grad_() for t in wrt]
    mag = _reference(*mags[:3], a, mags[3], None, 64 ** -0.5)
    mgrads = torch.autograd.grad(mag, mags, (do.abs().double(), torch.ones_like(rfinal)))
    growth = _growth(200, 64, 64, dtype)
    _check(out, ref, mag[0], dtype, growth, "out")
    _check(final, rfinal, mag[1], dtype, growth, "final state", state=True)
    for name, g, r, m in zip(("dq", "dk", "dv", "ds0"), grads, rgrads, mgrads):
        _check(g, r, m, dtype, growth, name, state=name == "ds0")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_padding_may_hold_anything(dtype):
    lengths = [130, 0, 77, 256]
    q, k, v, a, s0, n = _inputs(4, 256, 2, 2, 64, 64, dtype, 7, True, lengths)
    do = torch.randn(4, 256, 2, 64, device=DEV).to(dtype)
    results = []
    for junk in (0.0, float("nan"), float("inf")):
        qj, kj, vj, dj = (t.clone() for t in (q, k, v, do))
        for b, m in enumerate(lengths):
            for t in (qj, kj, vj, dj):
                t[b, m:] = junk
        for t in (qj, kj, vj):
            t.requires_grad_()
        out, final = F.linear_attention(qj, kj, vj, a, initial_state=s0, lengths=n)
        results.append((out, final, *torch.autograd.grad(out, (qj, kj, vj), dj)))
    for other in results[1:]:
        for x, y in zip(results[0], other):
            assert torch.equal(x, y)
    for t in (results[0][0], *results[0][2:]):
        for b, m in enumerate(lengths):
            assert not t[b, m:].any()
    assert torch.equal(results[0][1][1], s0[1])  # no token: the state passes through


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Head-major tensors, slices of one projection, misaligned rows, broadcast heads."""
    B, L, H, D = 2, 150, 3, 32
    q, k, v, a, _, _ = _inputs(B, L, H, H, D, D, dtype, 9)
    want = F.linear_attention(q, k, v, a)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    joined = torch.cat([t.flatten(-2) for t in (q, k, v)], -1)
    parts = [t.unflatten(-1, (H, D)) for t in joined.split(H * D, -1)]
    shifted = []
    for t in (q, k, v):
        flat = torch.empty(t.numel() + 1, device=DEV, dtype=dtype)
        flat[1:] = t.flatten()
        shifted.append(flat[1:].view(t.shape))
    assert shifted[0].data_ptr() % 16 != 0
    inner = [torch.stack([t, t], -1)[..., 0] for t in (q, k, v)]  # last axis not contiguous
    tol = 0 if dtype == torch.float32 else None
    for operands in (major, parts, shifted, inner):
        got = F.linear_attention(*operands, a)
        for g, w in zip(got, want):
            if tol == 0:
                assert torch.equal(g, w)
            else:
                ref = _reference(q, k, v, a, None, None, D ** -0.5)
                mag = _magnitudes(q, k, v, a, None, None, D ** -0.5)
                _check(got[0], ref[0], mag[0], dtype, _growth(L, D, D, dtype), "out")
                _check(got[1], ref[1], mag[1], dtype, _growth(L, D, D, dtype), "state", True)
    one = [t[:, :, :1] for t in (k, v)]
    wide = [t.expand(B, L, H, D) for t in one]  # stride zero over the heads
    for g, w in zip(F.linear_attention(q, *wide, a), F.linear_attention(q, *one, a)):
        assert torch.equal(g, w)


def test_gradient_of_expanded_output():
    """d_out of a plain sum has stride zero on every axis."""
    q, k, v, a, _, _ = _inputs(1, 70, 2, 2, 16, 16, torch.float32, 11)
    q.requires_grad_()
    (g,) = torch.autograd.grad(F.linear_attention(q, k, v, a)[0].sum(), q)
    (h,) = torch.autograd.grad(F.linear_attention(q, k, v, a)[0], q,
                               torch.ones(1, 70, 2, 16, device=DEV))
    assert torch.equal(g, h)


def test_state_gradient_alone():
    q, k, v, a, s0, _ = _inputs(1, 90, 2, 1, 24, 40, torch.float64, 13, True)
    for t in (k, v, s0):
        t.requires_grad_()
    final = F.linear_attention(q, k, v, a, initial_state=s0)[1]
    ref = _reference(q, k, v, a, s0, None, 24 ** -0.5)[1]
    w = torch.randn_like(final)
    for g, r in zip(torch.autograd.grad(final, (k, v, s0), w),
                    torch.autograd.grad(ref, (k, v, s0), w)):
        assert (g - r).abs().max() <= 1e-12 * r.abs().max()


def test_gradients_by_differences():
    q, k, v, a, s0, n = _inputs(2, 5, 4, 2, 3, 2, torch.float64, 15, True, [5, 3])
    for t in (q, k, v, s0):
        t.requires_grad_()
    assert torch.autograd.gradcheck(
        lambda *t: F.linear_attention(*t[:3], a, initial_state=t[3], lengths=n), (q, k, v, s0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeatable_and_other_stream(dtype):
    q, k, v, a, _, _ = _inputs(2, 2000, 4, 2, 64, 64, dtype, 17)
    do = torch.randn(2, 2000, 4, 64, device=DEV).to(dtype)

    def step():
        ts = [t.detach().requires_grad_() for t in (q, k, v)]
        out, final = F.linear_attention(*ts, a)
        return (out, final, *torch.autograd.grad(out, ts, do))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, again):
        assert torch.equal(x, y)


def test_empty_batch_and_empty_sequence():
    q, k, v, a, s0, _ = _inputs(2, 0, 2, 2, 8, 8, torch.float32, 0, True)
    s0.requires_grad_()
    out, final = F.linear_attention(q, k, v, a, initial_state=s0)
    assert out.shape == (2, 0, 2, 8) and torch.equal(final, s0)
    (g,) = torch.autograd.grad(final, s0, torch.ones_like(final))
    assert torch.equal(g, torch.ones_like(g))
    assert not F.linear_attention(q, k, v, a)[1].any()
    out, final = F.linear_attention(q[:0], k[:0], v[:0], a)
    assert out.shape == (0, 0, 2, 8) and final.shape == (0, 2, 8, 8)


# ------------------------------------------------------------------------------ single tokens


def _step_reference(q, k, v, a, state, scale):
    q, k, v, state = (t.double() for t in (q, k, v, state))
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    state = a.double().exp().view(1, -1, 1, 1) * state + k.unsqueeze(-1) * v.unsqueeze(-2)
    return scale * torch.einsum("bhd,bhde->bhe", q, state), state


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", [(1, 1, 1, 1, 1), (1, 4, 4, 64, 64), (3, 4, 2, 33, 7),
                                          (2, 6, 1, 128, 200), (70, 2, 2, 256, 256),
                                          (5, 3, 3, 16, 130)])
def test_step(B, H, Hk, Dk, Dv, dtype):
    torch.manual_seed(B + Dk)
    acc = torch.float64 if dtype == torch.float64 else torch.float32
    q = torch.randn(B, H, Dk, device=DEV).to(dtype)
    k = torch.randn(B, Hk, Dk, device=DEV).to(dtype)
    v = torch.randn(B, Hk, Dv, device=DEV).to(dtype)
    state = torch.randn(B, H, Dk, Dv, device=DEV, dtype=acc)
    a = _schedule(H).to(acc)
    a[0] = -float("inf")
    ref, rstate = _step_reference(q, k, v, a, state, 0.7)
    mag = _step_reference(q.abs(), k.abs(), v.abs(), a, state.abs(), 0.7)
    out = F.linear_attention_step(q, k, v, a, state, scale=0.7)
    unit = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    bound = (Dk + 8) * unit * mag[0] + ROUND[dtype] * ref.abs() + 2.0 ** -24 * (dtype in HALF)
    assert ((out.double() - ref).abs() <= bound).all()
    assert ((state.double() - rstate).abs() <= 4 * unit * mag[1]).all()


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_step_slots(index):
    torch.manual_seed(3)
    q, k = torch.randn(5, 2, 32, device=DEV), torch.randn(5, 2, 32, device=DEV)
    v = torch.randn(5, 2, 48, device=DEV)
    a = _schedule(2)
    pool = torch.randn(6, 2, 32, 48, device=DEV)
    before = pool.clone()
    far = 6 if index == torch.int32 else (1 << 40)
    slots = torch.tensor([4, -1, 0, far, 2], dtype=index, device=DEV)
    out = F.linear_attention_step(q, k, v, a, pool, slots=slots)
    live, used = [0, 2, 4], [4, 0, 2]
    dense = before[used].clone()
    want = F.linear_attention_step(q[live], k[live], v[live], a, dense)
    assert torch.equal(out[live], want) and not out[[1, 3]].any()
    assert torch.equal(pool[used], dense)
    assert torch.equal(pool[[1, 3, 5]], before[[1, 3, 5]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_steps_equal_the_whole(dtype):
    q, k, v, a, _, _ = _inputs(2, 140, 4, 2, 64, 64, dtype, 19)
    whole, last = F.linear_attention(q, k, v, a)
    out, state = F.linear_attention(q[:, :130], k[:, :130], v[:, :130], a)
    outs = [out]
    for t in range(130, 140):
        outs.append(F.linear_attention_step(q[:, t], k[:, t], v[:, t], a, state).unsqueeze(1))
    ref = _reference(q, k, v, a, None, None, 64 ** -0.5)
    mag = _magnitudes(q, k, v, a, None, None, 64 ** -0.5)
    growth = _growth(140, 64, 64, dtype)
    for got in (whole, torch.cat(outs, 1)):
        _check(got, ref[0], mag[0], dtype, growth, "out")
    for got in (last, state):
        _check(got, ref[1], mag[1], dtype, growth, "state", state=True)


def test_refusals():
    q, k, v, a, s0, n = _inputs(2, 8, 4, 2, 16, 16, torch.float32, 0, True, [8, 3])
    bad = [
        (ValueError, lambda: F.linear_attention(q, k[:, :7], v, a)),
        (ValueError, lambda: F.linear_attention(q, k, v[:, :, :1], a)),
        (ValueError, lambda: F.linear_attention(q[..., :8], k, v, a)),
        (ValueError, lambda: F.linear_attention(q[:, :, :3], k, v, a[:3])),
        (ValueError, lambda: F.linear_attention(q, k, v, a[:2])),
        (ValueError, lambda: F.linear_attention(q[0], k[0], v[0], a)),
        (TypeError, lambda: F.linear_attention(q, k.half(), v, a)),
        (TypeError, lambda: F.linear_attention(q.int(), k.int(), v.int(), a)),
        (ValueError, lambda: F.linear_attention(q, k, v, a, initial_state=s0[:1])),
        (ValueError, lambda: F.linear_attention(q, k, v, a, initial_state=s0.half())),
        (ValueError, lambda: F.linear_attention(q, k, v, a, lengths=n[:1])),
        (ValueError, lambda: F.linear_attention(q, k, v, a, lengths=n.float())),
        (ValueError, lambda: F.linear_attention(q, k, v, a.clone().requires_grad_())),
        (RuntimeError, lambda: F.linear_attention(q.cpu(), k.cpu(), v.cpu(), a.cpu())),
        (RuntimeError, lambda: F.linear_attention(q, k, v, a.cpu())),
        (ValueError, lambda: F.linear_attention(*(torch.zeros(1, 2, 1, 300, device=DEV),) * 3,
                                                a[:1])),
        (ValueError, lambda: F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, s0[:1])),
        (ValueError, lambda: F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a,
                                                     s0.transpose(2, 3))),
        (ValueError, lambda: F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a, s0,
                                                     slots=n[:1])),
        (RuntimeError, lambda: F.linear_attention_step(q[:, 0].clone().requires_grad_(), k[:, 0],
                                                       v[:, 0], a, s0)),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    lib = _lib.load()
    assert lib.fdwt_linattn_forward(None, *[None] * 9, 0, None) == 1
    q.requires_grad_()
    out, _ = F.linear_attention(q, k, v, a)
    with pytest.raises(RuntimeError):  # differentiable once
        (g,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
        g.sum().backward()


# ------------------------------------------------------------------------------ the layer


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decay_token_mixer(dtype):
    """Training step, prompt of uneven lengths in a pool of states, then single tokens."""
    torch.manual_seed(21)
    layer = F.DecayTokenMixer(96, num_heads=6, num_kv_heads=2).to(DEV)
    with torch.no_grad():
        layer.norm.bias.normal_()
    layer = layer.to(dtype)
    B, L = 3, 150
    x = torch.randn(B, L, 96, device=DEV).to(dtype).requires_grad_()
    y = layer(x)
    y.float().square().sum().backward()
    assert y.dtype == dtype and all(p.grad is not None for p in layer.parameters())

    def plain(x):
        P = {k: p.detach().double() for k, p in layer.named_parameters()}
        x = x.detach().double()
        c = x - x.mean(-1, keepdim=True)
        h = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5)
        h = h * P["norm.weight"] + P["norm.bias"]
        q, k, v = (h @ P["qkv_proj.weight"].T + P["qkv_proj.bias"]).split([96, 32, 32], -1)
        o, s = _reference(q.unflatten(-1, (6, 16)), k.unflatten(-1, (2, 16)),
                          v.unflatten(-1, (2, 16)), layer.log_decay(DEV), None, None, 0.25)
        return x + o.flatten(-2) @ P["out_proj.weight"].T + P["out_proj.bias"], s

    ref, rstate = plain(x)
    tol = 2e-5 if dtype == torch.float32 else 4 * ROUND[dtype]
    assert (y.double() - ref).square().mean().sqrt() <= tol * ref.square().mean().sqrt()
    # serving: prompts of 150, 149 and 1 tokens, then the rest token by token
    lengths = torch.tensor([150, 149, 1], device=DEV)
    with torch.no_grad():
        out, state = layer(x, lengths=lengths, return_state=True)
        pool = layer.init_state(5, DEV)
        slots = torch.tensor([3, 0, 4], device=DEV)
        pool[slots] = state
        token = layer.step(x[:, 149], pool, slots=torch.tensor([-1, 0, -1], device=DEV))
    assert (token[1].double() - ref[1, 149]).abs().max() <= 4 * tol * ref.abs().max()
    assert torch.equal(pool[3], state[0]) and torch.equal(pool[4], state[2])
    got = pool[0].double()
    assert (got - rstate[1]).abs().max() <= 8 * tol * rstate.abs().max()
    if dtype == torch.float32:  # causal: the past does not see the future
        z = x.detach().clone()
        z[:, 100:] = torch.randn_like(z[:, 100:])
        assert torch.equal(layer(z)[:, :100], y[:, :100])


def test_decay_token_mixer_refusals():
    with pytest.raises(ValueError):
        F.DecayTokenMixer(10, num_heads=4)
    with pytest.raises(ValueError):
        F.DecayTokenMixer(16, num_heads=4, num_kv_heads=3)
    layer = F.DecayTokenMixer(16, num_heads=4).to(DEV)
    with pytest.raises(ValueError):
        layer(torch.zeros(2, 16, device=DEV))
    with pytest.raises(ValueError):
        layer.step(torch.zeros(2, 1, 16, device=DEV), layer.init_state(2, DEV))
