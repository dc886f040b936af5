"""selective_scan, its gradients and its single-token form against the recurrence in 64 bits.

Tolerances, set from the arithmetic.  A decay e^(delta a) in 32 bits is off by a few roundings
times (1 + |delta a|) (the step's own, the product's, the exponential's 2 units), and a state is a
sum of products of decays: a token's share has the error of every decay since.  The sum of
magnitudes S_t = e^(delta a) S_{t-1} + |delta x b| therefore has with it an error E_t =
e^(delta a) (E_{t-1} + (1 + |delta a|) S_{t-1}) + |delta x b|, in units of ``GROWTH`` = 8
roundings, which the reference carries along; gradients have the same back in time, and sums over
states, channels and tokens add those of their terms (in short runs and trees, within the 8).  A
result rounded once to a type of unit roundoff u is off by u |result| more.
"""

import pytest
import torch

import pytorch_morlet_fdwt_b200 as F
from pytorch_morlet_fdwt_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64, F32, F16, BF16 = torch.float64, torch.float32, torch.float16, torch.bfloat16
ROUND = {F64: 2.0 ** -53, F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F64: 1e-300, F32: 2.0 ** -120, F16: 2.0 ** -24, BF16: 2.0 ** -120}
GROWTH = 8
NAMES = ("x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "initial")


def _acc(dtype):
    return 2.0 ** -53 if dtype == F64 else 2.0 ** -24


def _case(B, L, D, N, G=1, dtype=F32, gate=True, skip=True, bias=True, initial=True, lengths=None,
          softplus=True, seed=0):
    torch.manual_seed(seed)
    wide = F64 if dtype == F64 else F32

    def normal(*shape, to=dtype):
        return torch.randn(*shape, device=DEV).to(to)

    s = {"x": normal(B, L, D), "dt": normal(B, L, D), "b": normal(B, L, G, N),
         "c": normal(B, L, G, N)}
    s["a"] = -torch.exp(torch.randn(D, N, device=DEV)).to(wide)
    s["skip"] = normal(D, to=wide) if skip else None
    s["gate"] = normal(B, L, D) if gate else None
    s["dt_bias"] = (normal(D, to=wide) - 2) if bias else None
    if not softplus:
        s["dt"] = (s["dt"].abs() * 0.2).to(dtype)
        s["dt_bias"] = s["dt_bias"].abs() * 0.1 if bias else None
    s["initial"] = normal(B, D, N, to=wide) if initial else None
    s["lengths"] = None if lengths is None else torch.tensor(lengths, device=DEV, dtype=torch.int32)
    s["softplus"] = softplus
    return s


def _call(s):
    return F.selective_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], s["skip"], s["gate"],
                            s["dt_bias"], s["softplus"], s["initial"], s["lengths"])


def _reference(s, dy=None, df=None):
    """{name: (value, error in roundings)} of y and final, and with dy of the gradients."""
    x, dt, a, b, c = (s[k].detach().double() for k in ("x", "dt", "a", "b", "c"))
    B, L, D = x.shape
    G, N = b.shape[2:]
    zero = torch.zeros(D, device=DEV, dtype=F64)
    skip = zero if s["skip"] is None else s["skip"].detach().double()
    v = dt if s["dt_bias"] is None else dt + s["dt_bias"].detach().double()
    n = s["lengths"]
    count = torch.full((B,), L, device=DEV) if n is None else n.clamp(0, L)
    live = (torch.arange(L, device=DEV) < count.view(B, 1)).unsqueeze(-1)
    v = torch.where(live, v, 0.0)
    delta = torch.logaddexp(v, torch.zeros_like(v)) if s["softplus"] else v
    delta, x = torch.where(live, delta, 0.0), torch.where(live, x, 0.0)
    of = torch.arange(D, device=DEV) // (D // G)
    live4 = live.unsqueeze(-1)
    b, c = (torch.where(live4, t[:, :, of], 0.0) for t in (b, c))     # (B, L, D, N)
    h = torch.zeros(B, D, N, device=DEV, dtype=F64)
    if s["initial"] is not None:
        h = s["initial"].detach().double().clone()
    mag, err = h.abs(), torch.zeros_like(h)
    H, M, E = [h], [mag], [err]
    decay = torch.exp(delta.unsqueeze(-1) * a)
    rough = 1 + (delta.unsqueeze(-1) * a).abs()
    into = (delta * x).unsqueeze(-1) * b
    for t in range(L):
        h = decay[:, t] * h + into[:, t]
        err = decay[:, t] * (err + rough[:, t] * mag) + into[:, t].abs()
        mag = decay[:, t] * mag + into[:, t].abs()
        H.append(h), M.append(mag), E.append(err)
    H, M, E = (torch.stack(q, 1) for q in (H, M, E))
    p = (H[:, 1:] * c).sum(-1) + skip * x
    pe = ((E[:, 1:] + 2 * M[:, 1:]) * c.abs()).sum(-1) + (skip * x).abs()
    opened, opening, z = torch.ones_like(p), None, None
    if s["gate"] is not None:
        z = torch.where(live, s["gate"].detach().double(), 0.0)
        sg = torch.sigmoid(z)
        opened, opening = z * sg, sg * (1 + z * (1 - sg))
    size = opened.abs() * (1 + (0 if z is None else z.abs()))
    res = {"y": (p * opened, (pe + 2 * p.abs()) * size), "final": (H[:, -1], E[:, -1] + M[:, -1])}
    if dy is None:
        return res
    dy = torch.where(live, dy.double(), 0.0)
    dp, dpe = dy * opened, 2 * dy.abs() * size
    if z is not None:
        res["gate"] = (dy * p * opening, dy.abs() * (pe + 2 * p.abs()) * (1.2 + z.abs()))
    r = torch.zeros(B, D, N, device=DEV, dtype=F64) if df is None else df.double().clone()
    rm, re = r.abs(), torch.zeros_like(r)
    da, dae = torch.zeros_like(a), torch.zeros_like(a)
    out = {k: (torch.zeros_like(x), torch.zeros_like(x)) for k in ("x", "dt")}
    out |= {k: (torch.zeros_like(b), torch.zeros_like(b)) for k in ("b", "c")}
    slope = torch.sigmoid(v) if s["softplus"] else torch.ones_like(v)
    slope = torch.where(live, slope, 0.0)
    for t in range(L - 1, -1, -1):
        q, qe = dp[:, t].unsqueeze(-1), dpe[:, t].unsqueeze(-1)
        g = c[:, t] * q + r
        gm = (c[:, t] * q).abs() + rm
        ge = c[:, t].abs() * (q.abs() + qe) + re
        out["c"][0][:, t] = q * H[:, t + 1]
        out["c"][1][:, t] = q.abs() * (E[:, t + 1] + 2 * M[:, t + 1]) + qe * M[:, t + 1]
        dx_ = (delta[:, t] * x[:, t]).unsqueeze(-1)
        out["b"][0][:, t] = g * dx_
        out["b"][1][:, t] = (ge + 3 * gm) * dx_.abs()
        through = (g * b[:, t]).sum(-1)
        te = ((ge + 2 * gm) * b[:, t].abs()).sum(-1)
        r = decay[:, t] * g
        re, rm = decay[:, t] * (ge + rough[:, t] * gm), decay[:, t] * gm
        k = r * H[:, t]
        ke = rm * E[:, t] + (re + 2 * rm) * M[:, t]
        dl = delta[:, t].unsqueeze(-1)
        da += (dl * k).sum(0)
        dae += (dl * (ke + 2 * rm * M[:, t])).sum(0)
        out["x"][0][:, t] = delta[:, t] * through + skip * dp[:, t]
        out["x"][1][:, t] = delta[:, t] * (te + 2 * through.abs()) + skip.abs() * (dp + dpe)[:, t].abs()
        dd = (a * k).sum(-1) + x[:, t] * through
        de = (a.abs() * (ke + 2 * rm * M[:, t])).sum(-1) + x[:, t].abs() * (te + 2 * through.abs())
        out["dt"][0][:, t] = dd * slope[:, t]
        out["dt"][1][:, t] = (de + 2 * dd.abs()) * slope[:, t] * (1 + v[:, t].abs())
    res |= {"x": out["x"], "dt": out["dt"], "a": (da, dae)}
    for k in ("b", "c"):
        res[k] = tuple(t.view(B, L, G, D // G, N).sum(3) for t in out[k])
    res["skip"] = ((dp * x).sum((0, 1)), ((dp.abs() * 3 + dpe) * x.abs()).sum((0, 1)))
    res["dt_bias"] = (out["dt"][0].sum((0, 1)), (out["dt"][1] + 2 * out["dt"][0].abs()).sum((0, 1)))
    res["initial"] = (r, re + rm)
    return res


def _check(got, ref, dtype, what, acc=None):
    value, error = ref
    assert got.dtype == dtype and got.shape == value.shape, what
    bound = ROUND[dtype] * value.abs() + GROWTH * (acc or _acc(dtype)) * error + TINY[dtype]
    worst = ((got.double() - value).abs() / bound).max() if got.numel() else torch.zeros(())
    assert worst <= 1.0, f"{what}: {worst:.3g} of the tolerance"


def _forward_and_gradients(s, with_final=True):
    dtype = s["x"].dtype
    B, L, D = s["x"].shape
    if s["lengths"] is not None:  # padding may hold anything
        for i, n in enumerate(s["lengths"].tolist()):
            for k, bad in (("x", float("nan")), ("dt", float("inf")), ("b", float("-inf")),
                           ("c", float("nan")), ("gate", float("nan"))):
                if s[k] is not None:
                    s[k][i, max(0, n):] = bad
    leaves = [k for k in NAMES if s[k] is not None]
    for k in leaves:
        s[k].requires_grad_()
    before = _lib.launch_count()
    y, final = _call(s)
    assert _lib.launch_count() > before
    torch.manual_seed(7)
    dy = torch.randn(B, L, D, device=DEV).to(dtype)
    df = torch.randn_like(final) if with_final else None
    ref = _reference(s, dy, df)
    wide = final.dtype
    _check(y.detach(), ref["y"], dtype, "y", _acc(dtype))
    _check(final.detach(), ref["final"], wide, "final")
    with torch.no_grad():  # without gradients the same bits
        again = _call(s)
    assert torch.equal(again[0], y) and torch.equal(again[1], final)
    outs, gs = ((y, final), (dy, df)) if with_final else ((y,), (dy,))
    grads = torch.autograd.grad(outs, [s[k] for k in leaves], gs)
    for k, g in zip(leaves, grads):
        _check(g, ref[k], s[k].dtype, f"dL/d{k}", _acc(dtype))
    return y, final, grads


CASES = [  # B, L, D, N, G, options
    (1, 1, 1, 1, 1, {}), (1, 1, 8, 16, 1, {"initial": False}), (2, 2, 16, 16, 2, {}),
    (3, 7, 24, 3, 3, {"lengths": [7, 0, 1]}), (2, 8, 64, 4, 1, {"gate": False}),
    (2, 9, 40, 8, 1, {"skip": False}), (1, 17, 96, 16, 1, {"softplus": False}),
    (2, 37, 130, 12, 1, {"bias": False}), (4, 65, 66, 16, 3, {"lengths": [65, 0, 2, 64]}),
    (2, 100, 200, 17, 1, {}), (1, 130, 64, 32, 4, {"softplus": False, "bias": False}),
    (2, 77, 33, 64, 1, {"lengths": [-3, 999]}), (1, 50, 24, 100, 2, {}), (1, 33, 70, 128, 1, {}),
    (2, 300, 160, 16, 1, {"lengths": [299, 130]}), (1, 1500, 32, 16, 1, {}),
    (1, 700, 16, 5, 2, {"lengths": [650]}), (2, 0, 16, 4, 1, {}), (1, 260, 1024, 2, 1, {}),
    (1, 520, 72, 40, 3, {"gate": False, "skip": False, "initial": False})]


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("B,L,D,N,G,options", CASES)
def test_forward_and_gradients(B, L, D, N, G, options, dtype):
    _forward_and_gradients(_case(B, L, D, N, G, dtype, seed=L + N, **options))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,D", [(40, 24, 512), (5, 40, 4096), (160, 9, 130)])
def test_many_channels(B, L, D, dtype):
    """Enough blocks that a thread of the backward pass takes several channels."""
    _forward_and_gradients(_case(B, L, D, 16, 1, dtype, seed=B), with_final=False)


def test_gradients_against_differences():
    """fp64: central differences of step s are off by s^2 / 6 times a third derivative (here below
    1000) and 2^-53 / s of the values: 1e-7 of them at s = 1e-5."""
    for options in ({}, {"gate": False, "softplus": False, "lengths": [5, 2]}):
        s = _case(2, 5, 4, 3, 2, F64, **options)
        names = [k for k in NAMES if s[k] is not None]
        for k in names:
            s[k].requires_grad_()
        assert torch.autograd.gradcheck(
            lambda *t: _call(s | dict(zip(names, t))), [s[k] for k in names], eps=1e-5, atol=1e-6)


@pytest.mark.parametrize("dtype,N", [(F32, 16), (BF16, 16), (BF16, 7), (F64, 32)])
def test_a_cut_sequence_is_the_whole(dtype, N):
    """Calls that hand the state on, and single tokens, against the recurrence as one call."""
    s = _case(3, 40, 72, N, 2, dtype)
    ref = _reference(s)

    def part(i, j, state):
        return _call(s | {k: None if s[k] is None else s[k][:, i:j]
                          for k in ("x", "dt", "b", "c", "gate")} | {"initial": state})

    for cut in (1, 8, 17):
        y1, h = part(0, cut, s["initial"])
        y2, h = part(cut, 40, h)
        _check(torch.cat([y1, y2], 1), ref["y"], dtype, "y", _acc(dtype))
        _check(h, ref["final"], h.dtype, "final")
    y, h = part(0, 30, s["initial"])
    ys = [y]
    for t in range(30, 40):
        ys.append(F.selective_scan_step(s["x"][:, t], s["dt"][:, t], s["a"], s["b"][:, t],
                                        s["c"][:, t], h, s["skip"], s["gate"][:, t], s["dt_bias"],
                                        True).unsqueeze(1))
    _check(torch.cat(ys, 1), ref["y"], dtype, "y", _acc(dtype))
    _check(h, ref["final"], h.dtype, "final")


@pytest.mark.parametrize("dtype", [F32, F64, F16, BF16])
@pytest.mark.parametrize("D,N,G", [(1, 1, 1), (64, 16, 1), (33, 12, 3), (130, 7, 2), (40, 128, 1),
                                   (2048, 16, 1), (96, 64, 4), (50, 2, 1)])
def test_step_with_slots(D, N, G, dtype):
    for options in ({}, {"gate": False, "skip": False, "softplus": False}):
        s = _case(5, 1, D, N, G, dtype, initial=False, seed=D, **options)
        wide = F64 if dtype == F64 else F32
        pool = torch.randn(7, D, N, device=DEV, dtype=wide)
        before = pool.clone()
        slots = torch.tensor([6, -1, 0, 7, 3], device=DEV)
        token = {k: None if s[k] is None else s[k][:, 0] for k in ("x", "dt", "b", "c", "gate")}
        y = F.selective_scan_step(token["x"], token["dt"], s["a"], token["b"], token["c"], pool,
                                  s["skip"], token["gate"], s["dt_bias"], s["softplus"], slots)
        touched = []
        for i, slot in enumerate(slots.tolist()):
            if not 0 <= slot < 7:
                assert not y[i].any()
                continue
            touched.append(slot)
            one = {k: t[i:i + 1] if k in token and t is not None else t for k, t in s.items()}
            ref = _reference(one | {"initial": before[slot:slot + 1]})
            _check(y[i:i + 1], tuple(t[:, 0] for t in ref["y"]), dtype, "y", _acc(dtype))
            _check(pool[slot:slot + 1], ref["final"], wide, "state")
        rest = [i for i in range(7) if i not in touched]
        assert torch.equal(pool[rest], before[rest])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_offsets(dtype):
    """Inputs that are slices of projections' results, at any offset, and a gradient of any
    strides."""
    torch.manual_seed(1)
    s = _case(2, 50, 64, 16, 1, dtype)
    wide = torch.randn(2, 50, 300, device=DEV).to(dtype)
    dy = torch.randn(2, 64, 50, device=DEV).to(dtype).transpose(1, 2)
    for begin in (0, 1, 8, 33):
        one = s | {"x": wide[..., begin:begin + 64], "gate": wide[..., begin + 64:begin + 128],
                   "dt": wide[..., begin + 128:begin + 192],
                   "b": wide[..., begin + 192:begin + 208].unsqueeze(2),
                   "c": wide[..., begin + 208:begin + 224].unsqueeze(2)}
        names = ("x", "dt", "b", "c", "gate")
        one |= {k: one[k].detach().requires_grad_() for k in names}
        y, f = _call(one)
        ref = _reference(one, dy)
        _check(y.detach(), ref["y"], dtype, "y", _acc(dtype))
        _check(f.detach(), ref["final"], F32, "final")
        for k, g in zip(names, torch.autograd.grad(y, [one[k] for k in names], dy)):
            _check(g, ref[k], dtype, f"dL/d{k}", _acc(dtype))
        rows = {k: one[k].detach()[:, 3] for k in names}
        h = s["initial"].clone()
        y = F.selective_scan_step(rows["x"], rows["dt"], s["a"], rows["b"], rows["c"], h, s["skip"],
                                  rows["gate"], s["dt_bias"], True)
        ref = _reference(one | {k: one[k][:, 3:4] for k in names})
        _check(y, tuple(t[:, 0] for t in ref["y"]), dtype, "y", _acc(dtype))
        _check(h, ref["final"], F32, "state")


def test_last_axes_that_are_not_contiguous():
    """Inputs with another axis contiguous, or expanded over the channels or states: as their copies."""
    s = _case(2, 21, 24, 8, 1, F32)
    whole = _call(s)
    turned = s | {k: s[k].transpose(1, -1).contiguous().transpose(1, -1)
                  for k in ("x", "dt", "gate", "b", "c")}
    assert all(torch.equal(p, q) for p, q in zip(_call(turned), whole))
    wide = s | {"dt": s["dt"][..., :1].expand(2, 21, 24), "b": s["b"][..., :1].expand(2, 21, 1, 8)}
    copy = s | {k: wide[k].contiguous() for k in ("dt", "b")}
    assert all(torch.equal(p, q) for p, q in zip(_call(wide), _call(copy)))
    one = {k: t[:, 4] if k in ("x", "dt", "b", "c", "gate") else t for k, t in s.items()}
    states = [s["initial"].clone(), s["initial"].clone()]
    outs = [F.selective_scan_step(f(one["x"]), one["dt"], s["a"], f(one["b"]), one["c"], h, s["skip"],
                                  f(one["gate"]), s["dt_bias"], True)
            for f, h in zip((lambda t: t.transpose(0, -1).contiguous().transpose(0, -1), lambda t: t),
                            states)]
    assert torch.equal(*outs) and torch.equal(*states)


def test_parameters_in_16_bits_are_taken_in_32():
    s = _case(2, 20, 32, 8, 1, BF16)
    low = s | {k: s[k].to(BF16).requires_grad_() for k in ("a", "skip", "dt_bias")}
    high = low | {k: low[k].detach().float().requires_grad_() for k in ("a", "skip", "dt_bias")}
    y, _ = _call(low)
    z, _ = _call(high)
    assert torch.equal(y, z)
    dy = torch.randn_like(y)
    for k in ("a", "skip", "dt_bias"):
        g, = torch.autograd.grad(y, low[k], dy, retain_graph=True)
        w, = torch.autograd.grad(z, high[k], dy, retain_graph=True)
        assert g.dtype == BF16 and torch.equal(g, w.to(BF16))


@pytest.mark.parametrize("L", [60, 700])
def test_infinities_and_nan_reach_no_earlier_token(L):
    s = _case(1, L, 48, 16, 1, F32, initial=False)
    want = _call(s)[0]
    for name, at in (("x", L // 2), ("dt", L // 2), ("gate", L // 2), ("b", L // 2), ("c", L // 2)):
        for bad in (float("nan"), float("inf")):
            t = s[name].clone()
            if name in ("b", "c"):
                t[0, at, 0, 3] = bad
            else:
                t[0, at, 5] = bad
            y = _call(s | {name: t})[0]
            assert torch.equal(y[:, :at], want[:, :at])
            if name in ("x", "dt", "gate"):  # nor another channel
                keep = [c for c in range(48) if c != 5]
                assert torch.equal(y[..., keep], want[..., keep])


def test_rates_of_minus_infinity_forget():
    s = _case(2, 30, 16, 4, 1, F32, lengths=[30, 11])
    s["a"][:, 1] = float("-inf")
    y, final = _call(s)
    much = s | {"a": s["a"].clamp(min=-1e30)}
    assert torch.isfinite(y).all() and torch.isfinite(final).all()
    z, last = _call(much)
    assert torch.equal(y, z) and torch.equal(final, last)


def test_steps_of_zero_keep_the_state():
    """A step of zero, and padding, leave a state as it is, bit by bit, over any number of tokens."""
    for dtype in (F32, F64, BF16):
        s = _case(2, 600, 40, 16, 1, dtype, softplus=False, bias=False, lengths=[600, 1])
        s["dt"].zero_()
        _, final = _call(s)
        assert torch.equal(final, s["initial"])
        for _ in range(3):
            F.selective_scan_step(s["x"][:, 0], s["dt"][:, 0], s["a"], s["b"][:, 0], s["c"][:, 0], final)
        assert torch.equal(final, s["initial"])


def test_streams_graphs_and_workspaces():
    """Another stream; two captured forward and backward passes replayed in turn."""
    cases = [_case(1, 900, 64, 16, 1, BF16, seed=i) for i in range(2)]
    names = [k for k in NAMES if cases[0][k] is not None]
    for s in cases:
        for k in names:
            s[k].requires_grad_()
    dy = torch.randn(1, 900, 64, device=DEV).to(BF16)

    def step(s):
        y, f = _call(s)
        return (y.detach(), f.detach(), *torch.autograd.grad(y, [s[k] for k in names], dy))

    want = [step(s) for s in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(cases[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, held = [], []
    for s in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(s))
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for h, w in zip(held, want):
        assert all(torch.equal(a, b) for a, b in zip(h, w))


def test_repeated_calls_give_the_same_bits():
    s = _case(3, 400, 300, 16, 2, BF16, lengths=[400, 31, 399])
    first = _forward_and_gradients(s)
    y, f = _call(s)
    assert torch.equal(y, first[0]) and torch.equal(f, first[1])


def test_autograd_manners():
    s = _case(2, 9, 16, 4)
    state = s["initial"].clone()
    s["x"].requires_grad_()
    y, _ = _call(s | {"initial": state})
    args = (s["x"][:, 0], s["dt"][:, 0], s["a"], s["b"][:, 0], s["c"][:, 0])
    with pytest.raises(RuntimeError, match="no gradient"):
        F.selective_scan_step(*args, state)
    with torch.no_grad():
        F.selective_scan_step(*args, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, final = _call(s)
    g, = torch.autograd.grad(final.sum(), s["x"], retain_graph=True)
    both, = torch.autograd.grad((y, final), s["x"], (torch.zeros_like(y), torch.ones_like(final)))
    assert torch.equal(g, both)
    with torch.inference_mode():
        F.selective_scan_step(*(t.detach().clone() for t in args), s["initial"].clone())


def test_refusals():
    s = _case(2, 9, 16, 4)
    bad = [({"x": s["x"][0]}, ValueError, "B, L, D"), ({"dt": s["dt"][:, :3]}, ValueError, "dt"),
           ({"gate": s["gate"][..., :3]}, ValueError, "gate"), ({"b": s["b"][:, :, 0]}, ValueError, "G, N"),
           ({"c": s["c"][..., :2]}, ValueError, "G, N"), ({"a": s["a"][:3]}, ValueError, "a must"),
           ({"dt": s["dt"].half()}, TypeError, "one type"), ({"skip": s["skip"][:2]}, ValueError, "skip"),
           ({"dt_bias": s["dt_bias"].long()}, ValueError, "dt_bias"),
           ({"initial": s["initial"].double()}, ValueError, "state"),
           ({"lengths": torch.ones(3, device=DEV, dtype=torch.int32)}, ValueError, "lengths"),
           ({"x": s["x"].cpu()}, RuntimeError, "CUDA")]
    for change, error, match in bad:
        with pytest.raises(error, match=match):
            _call(s | change)
    wide = torch.randn(2, 9, 1, 129, device=DEV)
    with pytest.raises(ValueError, match="128"):
        _call(s | {"b": wide, "c": wide, "a": torch.zeros(16, 129, device=DEV)})
    three = torch.randn(2, 9, 3, 4, device=DEV)
    with pytest.raises(ValueError, match="multiple"):
        _call(s | {"b": three, "c": three})
    args = [s[k][:, 0] if k != "a" else s[k] for k in ("x", "dt", "a", "b", "c")]
    with pytest.raises(ValueError, match="state"):
        F.selective_scan_step(*args, s["initial"][:1].clone())
    with pytest.raises(ValueError, match="contiguous"):
        F.selective_scan_step(*args, s["initial"].transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(ValueError, match="slots"):
        F.selective_scan_step(*args, s["initial"], slots=torch.ones(2, device=DEV))
