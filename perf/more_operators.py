"""What is measured of the selective token mixer's operators: root-mean-square norm with the
residual's addition (and an output in 8 bits), the short causal convolution, and the selective
state space scan, over whole sequences and for single tokens.

Every case is a dict of plain values; ``op`` says which operator it calls:

* ``norm``        ``rms_norm`` of ``(rows, dim)`` with the residual added
* ``norm_8bit``   ``rms_norm_quantized`` of the same: e4m3 values with scales
* ``norm_train``  ``rms_norm`` with its gradients (input, residual, weight)
* ``conv``        ``causal_conv1d`` over whole sequences, with the state after them
* ``conv_train``  the same with its gradients (input, weight, bias)
* ``conv_step``   ``causal_conv1d_step``: one token for every sequence, states updated in place
* ``scan``        ``selective_scan`` over whole sequences, with the state after them
* ``scan_train``  the same with its gradients (all inputs)
* ``scan_step``   ``selective_scan_step``: one token for every sequence, states updated in place

``run`` computes a case in elementary torch operations in 32 bits, or, with ``own`` set, through
the package's public functions.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6


# ------------------------------------------------------------------------------- the cases


def _norm(op, rows, dim, dtype, residual=True, group=0):
    return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual,
            "group": group}


def _conv(op, batch, length, dim, width, dtype, silu=True, ragged=False, initial=False):
    return {"op": op, "batch": batch, "length": length, "dim": dim, "width": width,
            "dtype": dtype, "silu": silu, "ragged": ragged, "initial": initial}


def _scan(op, batch, length, dim, states, groups, dtype, gate=True, ragged=False, initial=False):
    return {"op": op, "batch": batch, "length": length, "dim": dim, "states": states,
            "groups": groups, "dtype": dtype, "gate": gate, "ragged": ragged, "initial": initial}


def _conv_step(batch, dim, width, dtype, pool):
    return {"op": "conv_step", "batch": batch, "dim": dim, "width": width, "dtype": dtype,
            "silu": True, "pool": pool}


def _scan_step(batch, dim, states, groups, dtype, pool):
    return {"op": "scan_step", "batch": batch, "dim": dim, "states": states, "groups": groups,
            "dtype": dtype, "gate": True, "pool": pool}


def listed():
    cases = {
        # the norm before one decoded token of a few sequences: latency
        "norm_tokens": _norm("norm", 4, 256, "bf16"),
        # a prompt batch whose next product runs in 8 bits, scales for groups of 128
        "norm_8bit_groups": _norm("norm_8bit", 32768, 2048, "bf16", True, 128),
        # a large training batch of a wide model
        "norm_train_large": _norm("norm_train", 65536, 2048, "bf16"),
        # prompts of different lengths (an empty one among them) continued from states, full
        # precision, an odd width
        "conv_ragged_f32": _conv("conv", 5, 3001, 1001, 3, "f32", True, True, True),
        # a training step's convolution
        "conv_train_wide": _conv("conv_train", 4, 4096, 2048, 4, "bf16"),
        # one token for each of a pool of sequences: latency
        "conv_step_pool": _conv_step(240, 512, 4, "bf16", 256),
        # a short question: latency
        "scan_short": _scan("scan", 1, 37, 512, 16, 1, "bf16"),
        # the token mixers' shape (8, 4096, 256), inner width 512
        "scan_mixer": _scan("scan", 8, 4096, 512, 16, 1, "bf16"),
        # one long document
        "scan_long": _scan("scan", 1, 65536, 2048, 16, 1, "bf16"),
        # prompts of different lengths continued from states, full precision, channel groups,
        # uneven sizes
        "scan_ragged_f32": _scan("scan", 5, 1537, 690, 12, 3, "f32", False, True, True),
        # a training step's scan
        "scan_train_wide": _scan("scan_train", 4, 4096, 2048, 16, 1, "bf16"),
        # one token for each of a full pool of sequences
        "scan_step_pool": _scan_step(240, 2048, 16, 1, "bf16", 256),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def _width(rng, low, high):
    dim = _log_int(rng, low, high)
    return dim if rng.random() < 0.4 else max(low, dim // 64 * 64)


def draw(rng: random.Random):
    op = rng.choice(["norm", "norm_8bit", "norm_train", "conv", "conv_train", "conv_step",
                     "scan", "scan", "scan_train", "scan_train", "scan_step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("norm"):
        group = 0
        dim = _width(rng, 64, 8192)
        if op == "norm_8bit" and rng.random() < 0.6:
            group = rng.choice([32, 64, 128])
            dim = max(group, dim // group * group)
        most = min(65536, 2 ** 26 // dim)
        return _norm(op, _log_int(rng, 1, most), dim, dtype, rng.random() < 0.8, group)
    if op == "conv_step":
        batch = _log_int(rng, 1, 240)
        return _conv_step(batch, _width(rng, 64, 4096), rng.randrange(2, 6), dtype,
                          0 if rng.random() < 0.5 else batch + rng.randrange(1, 17))
    if op.startswith("conv"):
        dim = _width(rng, 64, 4096)
        batch = _log_int(rng, 1, 16)
        length = _log_int(rng, 1, min(65536, 2 ** 25 // dim) // batch)
        return _conv(op, batch, length, dim, rng.choice([2, 3, 4, 4, 4, 5]), dtype,
                     rng.random() < 0.8, rng.random() < 0.4, rng.random() < 0.4)
    states = rng.choice([8, 12, 16, 16, 16, 16, 32, 64])
    groups = rng.choice([1, 1, 1, 2, 4])
    dim = groups * max(16, _width(rng, 64, 2048) // groups)
    if op == "scan_step":
        batch = _log_int(rng, 1, 240)
        return _scan_step(batch, dim, states, groups, dtype,
                          0 if rng.random() < 0.5 else batch + rng.randrange(1, 17))
    batch = _log_int(rng, 1, 16)
    elements = 2 ** (30 if op == "scan" else 28)
    length = _log_int(rng, 1, min(65536, elements // (dim * states)) // batch)
    return _scan(op, batch, length, dim, states, groups, dtype, rng.random() < 0.7,
                 rng.random() < 0.4, rng.random() < 0.4)


# ------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device=device) * scale).to(to)

    def uniform(*shape, low=0.0, high=1.0):
        return low + (high - low) * torch.rand(*shape, generator=gen, device=device)

    state = {"case": case}
    if op.startswith("norm"):
        rows, dim = case["rows"], case["dim"]
        # a residual stream with a few strong channels, and a layer's answer to it
        strong = 1 + 4 * (uniform(dim) < 0.02)
        state["x"] = normal(rows, dim)
        state["residual"] = None
        if case["residual"]:
            state["residual"] = (3 * strong * torch.randn(rows, dim, generator=gen,
                                                          device=device)).to(dtype)
        state["weight"] = (1 + 0.1 * torch.randn(dim, generator=gen, device=device)).to(dtype)
        if op == "norm_train":
            state["dy"] = normal(rows, dim)
            state["dtotal"] = normal(rows, dim) if case["residual"] else None
            for key in ("x", "residual", "weight"):
                if state[key] is not None:
                    state[key].requires_grad_()
        return state

    batch, dim = case["batch"], case["dim"]
    state["slots"] = state["lengths"] = state["initial"] = None
    if op.endswith("step"):
        rows = case["pool"] or batch
        if case["pool"]:
            order = torch.randperm(rows, generator=gen, device=device)
            state["slots"] = order[:batch].to(torch.int32)
        lead = (batch,)
    else:
        lead = (batch, case["length"])
        if case["ragged"]:
            lengths = torch.randint(0, case["length"] + 1, (batch,), generator=gen, device=device)
            lengths[0] = case["length"]
            if batch > 1:
                lengths[-1] = 0
            state["lengths"] = lengths.to(torch.int32)
    state["x"] = normal(*lead, dim)

    if op.startswith("conv"):
        width = case["width"]
        state["weight"] = normal(dim, width, scale=width ** -0.5)
        state["bias"] = normal(dim, scale=0.1)
        if op == "conv_step":
            state["state"] = normal(rows, width - 1, dim)
            return state
        if case["initial"]:
            state["initial"] = normal(batch, width - 1, dim)
        if op == "conv_train":
            state["dy"] = normal(*lead, dim)
            for key in ("x", "weight", "bias"):
                state[key].requires_grad_()
        return state

    states, groups = case["states"], case["groups"]
    # rates 1..states for every channel and steps from 1/1000 to 1/10, as such layers start with
    state["a"] = -(torch.arange(1, states + 1, device=device, dtype=torch.float32)
                   * uniform(dim, 1, low=0.8, high=1.25))
    size = torch.exp(uniform(dim, low=math.log(1e-3), high=math.log(1e-1)))
    state["dt_bias"] = torch.log(torch.expm1(size))
    state["dt"] = normal(*lead, dim, scale=0.5)
    state["b"], state["c"] = normal(*lead, groups, states), normal(*lead, groups, states)
    state["skip"] = 1 + normal(dim, scale=0.1, to=torch.float32)
    state["gate"] = normal(*lead, dim) if case["gate"] else None
    if op == "scan_step":
        state["state"] = normal(rows, dim, states, scale=0.5, to=torch.float32)
        return state
    if case["initial"]:
        state["initial"] = normal(batch, dim, states, scale=0.5, to=torch.float32)
    if op == "scan_train":
        state["dy"] = normal(*lead, dim)
        for key in _scan_inputs(state):
            state[key].requires_grad_()
    return state


def _scan_inputs(state):
    """The inputs that a training step of the scan differentiates, in the order of its result."""
    names = ("x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "initial")
    return [name for name in names if state[name] is not None]


# ------------------------------------------------------------------------------- plain forms


def _plain_norm(state):
    """The sum in the inputs' type, and its norm in 32 bits."""
    x = state["x"]
    total = x
    if state["residual"] is not None:
        total = (x.float() + state["residual"].float()).to(x.dtype)
    h = total.float()
    rstd = (h.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    h = h * rstd
    return total, h, rstd, h * state["weight"].float()


def _run_plain_norm(state):
    op, x = state["case"]["op"], state["x"]
    total, h, rstd, y = _plain_norm(state)
    totals = [] if state["residual"] is None else [total]
    if op == "norm":
        return [y.to(x.dtype), *totals]
    if op == "norm_8bit":
        rows, dim = y.shape
        groups = y.view(rows, -1, state["case"]["group"] or dim)
        scale = groups.abs().amax(-1, keepdim=True) / 448.0
        scale = torch.where(scale > 0, scale, 1.0)
        q = (groups / scale).to(torch.float8_e4m3fn)
        return [q.view(rows, dim), scale.squeeze(-1), *totals]
    dy = state["dy"].float()
    g = dy * state["weight"].float()
    dx = rstd * (g - h * (g * h).mean(-1, keepdim=True))
    if state["dtotal"] is not None:
        dx = dx + state["dtotal"].float()
    dx = dx.to(x.dtype)
    dw = (dy * h).sum(0).to(x.dtype)
    return [y.to(x.dtype), *totals, dx, *([dx] if totals else []), dw]


def _valid(state, length):
    """(B, L, 1): which tokens count; None where all do."""
    lengths = state["lengths"]
    if lengths is None:
        return None
    t = torch.arange(length, device=lengths.device)
    return (t < lengths.view(-1, 1)).unsqueeze(-1)


def _silu_and_slope(p):
    s = 1 / (1 + torch.exp(-p))
    return p * s, s * (1 + p * (1 - s))


def _run_plain_conv(state):
    case = state["case"]
    x, weight, bias = (state[key].detach() for key in ("x", "weight", "bias"))
    dtype, width = x.dtype, case["width"]
    b, length, dim = x.shape
    before = state["initial"]
    if before is None:
        before = x.new_zeros(b, width - 1, dim)
    valid = _valid(state, length)
    tokens = x if valid is None else torch.where(valid, x, 0.0)
    whole = torch.cat([before, tokens], 1)
    windows = whole.float().unfold(1, width, 1)                  # (B, L, D, W)
    p = (windows * weight.float()).sum(-1) + bias.float()
    y, slope = _silu_and_slope(p) if case["silu"] else (p, torch.ones_like(p))
    if valid is not None:
        y = torch.where(valid, y, 0.0)
    n = state["lengths"]
    n = torch.full((b,), length, device=x.device) if n is None else n
    last = n.view(b, 1) + torch.arange(width - 1, device=x.device)
    final = whole.gather(1, last.long().unsqueeze(-1).expand(b, width - 1, dim))
    if case["op"] == "conv":
        return [y.to(dtype), final]
    dp = state["dy"].float() * slope
    if valid is not None:
        dp = torch.where(valid, dp, 0.0)
    after = torch.cat([dp, dp.new_zeros(b, width - 1, dim)], 1).unfold(1, width, 1)
    dx = (after * weight.float().flip(1)).sum(-1)
    if valid is not None:
        dx = torch.where(valid, dx, 0.0)
    dw = (dp.unsqueeze(-1) * windows).sum((0, 1))
    return [y.to(dtype), final, dx.to(dtype), dw.to(dtype), dp.sum((0, 1)).to(dtype)]


def _run_plain_conv_step(state):
    x, pool, slots = state["x"], state["state"], state["slots"]
    current = pool if slots is None else pool[slots.long()]
    window = torch.cat([current, x.unsqueeze(1)], 1)             # (B, W, D)
    p = (window.float() * state["weight"].float().T).sum(1) + state["bias"].float()
    if slots is None:
        pool.copy_(window[:, 1:])
    else:
        pool[slots.long()] = window[:, 1:]
    return [_silu_and_slope(p)[0].to(x.dtype), pool]


def _recurrence(decay, update):
    """h_t = decay_t h_{t-1} + update_t along the second axis, h_{-1} = 0, by doubling: after a
    round, entry t holds what the last 2, 4, 8, ... tokens up to t come to."""
    length, reach = update.shape[1], 1
    while reach < length:
        joined = update.clone()
        joined[:, reach:].addcmul_(decay[:, reach:], update[:, :-reach])
        update = joined
        if 2 * reach < length:
            joined = decay.clone()
            joined[:, reach:].mul_(decay[:, :-reach])
            decay = joined
        reach *= 2
    return update


def _steps(state):
    """The sizes of the steps: log(1 + e^v), v = dt + dt_bias, and their slope."""
    v = state["dt"].detach().float() + state["dt_bias"].detach()
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs())), 1 / (1 + torch.exp(-v))


def _channels(t, dim):
    """(..., G, N) for each channel: (..., D, N) in 32 bits."""
    return t.detach().float().repeat_interleave(dim // t.shape[-2], dim=-2)


def _run_plain_scan(state):
    case = state["case"]
    train = case["op"] == "scan_train"
    x, a, skip = (state[key].detach() for key in ("x", "a", "skip"))
    dtype = x.dtype
    bsz, length, dim = x.shape
    x = x.float()
    delta, slope = _steps(state)
    valid = _valid(state, length)
    if valid is not None:
        delta, x = torch.where(valid, delta, 0.0), torch.where(valid, x, 0.0)
    b, c = _channels(state["b"], dim), _channels(state["c"], dim)
    if valid is not None:
        b, c = torch.where(valid.unsqueeze(-1), b, 0.0), torch.where(valid.unsqueeze(-1), c, 0.0)
    decay = torch.exp(delta.unsqueeze(-1) * a)                   # (B, L, D, N)
    update = (delta * x).unsqueeze(-1) * b
    start = state["initial"]
    if start is not None:
        start = start.detach()
        update[:, 0] += decay[:, 0] * start
    h = _recurrence(decay, update)
    p = (h * c).sum(-1) + skip * x
    y = p
    if state["gate"] is not None:
        gate = state["gate"].detach().float()
        if valid is not None:
            gate = torch.where(valid, gate, 0.0)
        opened, opening = _silu_and_slope(gate)
        y = p * opened
    final = h[:, -1].clone()
    if not train:
        return [y.to(dtype), final]

    dy = state["dy"].float()
    if valid is not None:
        dy = torch.where(valid, dy, 0.0)
    dp = dy
    grads = {}
    if state["gate"] is not None:
        dp, grads["gate"] = dy * opened, (dy * p * opening).to(dtype)
    # the adjoint recurrence back in time
    later = torch.cat([decay[:, 1:], torch.ones_like(decay[:, :1])], 1)
    g = _recurrence(later.flip(1), (dp.unsqueeze(-1) * c).flip(1)).flip(1)
    first = torch.zeros_like(h[:, :1]) if start is None else start.unsqueeze(1)
    kept = g * decay * torch.cat([first, h[:, :-1]], 1)
    if start is not None:
        grads["initial"] = g[:, 0] * decay[:, 0]
    through = (g * b).sum(-1)
    ddelta = ((kept * a).sum(-1) + through * x) * slope
    groups, states = case["groups"], case["states"]
    grads["a"] = (kept * delta.unsqueeze(-1)).sum((0, 1))
    grads["x"] = (through * delta + skip * dp).to(dtype)
    grads["dt"] = ddelta.to(dtype)
    grads["dt_bias"] = ddelta.sum((0, 1))
    grads["skip"] = (dp * x).sum((0, 1))
    shape = (bsz, length, groups, dim // groups, states)
    grads["b"] = (g * (delta * x).unsqueeze(-1)).view(shape).sum(3).to(dtype)
    grads["c"] = (h * dp.unsqueeze(-1)).view(shape).sum(3).to(dtype)
    return [y.to(dtype), final, *(grads[key] for key in _scan_inputs(state))]


def _run_plain_scan_step(state):
    x = state["x"].float()
    dim = x.shape[1]
    delta = _steps(state)[0]
    pool, slots = state["state"], state["slots"]
    h = pool if slots is None else pool[slots.long()]
    h = (torch.exp(delta.unsqueeze(-1) * state["a"]) * h
         + (delta * x).unsqueeze(-1) * _channels(state["b"], dim))
    p = (h * _channels(state["c"], dim)).sum(-1) + state["skip"] * x
    if slots is None:
        pool.copy_(h)
    else:
        pool[slots.long()] = h
    return [(p * _silu_and_slope(state["gate"].float())[0]).to(state["x"].dtype), pool]


def _run_plain(state):
    op = state["case"]["op"]
    if op.startswith("norm"):
        return _run_plain_norm(state)
    if op == "conv_step":
        return _run_plain_conv_step(state)
    if op == "scan_step":
        return _run_plain_scan_step(state)
    return _run_plain_conv(state) if op.startswith("conv") else _run_plain_scan(state)


# ------------------------------------------------------------------------------- own kernels


def _run_own(state):
    import pytorch_morlet_fdwt_b200 as fdwt

    case = state["case"]
    op = case["op"]
    if op == "norm":
        out = fdwt.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=_EPS)
        return [out] if state["residual"] is None else list(out)
    if op == "norm_8bit":
        return list(fdwt.rms_norm_quantized(state["x"], state["weight"],
                                            residual=state["residual"], eps=_EPS,
                                            group_size=case["group"] or None))
    if op == "norm_train":
        out = fdwt.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=_EPS)
        if state["residual"] is None:
            grads = torch.autograd.grad(out, (state["x"], state["weight"]), state["dy"])
            return [out.detach(), *grads]
        grads = torch.autograd.grad(out, (state["x"], state["residual"], state["weight"]),
                                    (state["dy"], state["dtotal"]))
        return [*(o.detach() for o in out), *grads]
    if op == "conv_step":
        out = fdwt.causal_conv1d_step(state["x"], state["weight"], state["state"], state["bias"],
                                      activation="silu", slots=state["slots"])
        return [out, state["state"]]
    if op.startswith("conv"):
        inputs = (state["x"], state["weight"], state["bias"])
        out, final = fdwt.causal_conv1d(*inputs, activation="silu" if case["silu"] else None,
                                        initial_state=state["initial"], lengths=state["lengths"])
        if op == "conv":
            return [out, final]
        return [out.detach(), final.detach(), *torch.autograd.grad(out, inputs, state["dy"])]
    tokens = [state[key] for key in ("x", "dt", "a", "b", "c")]
    if op == "scan_step":
        out = fdwt.selective_scan_step(*tokens, state["state"], skip=state["skip"],
                                       gate=state["gate"], dt_bias=state["dt_bias"],
                                       dt_softplus=True, slots=state["slots"])
        return [out, state["state"]]
    out, final = fdwt.selective_scan(*tokens, skip=state["skip"], gate=state["gate"],
                                     dt_bias=state["dt_bias"], dt_softplus=True,
                                     initial_state=state["initial"], lengths=state["lengths"])
    if op == "scan":
        return [out, final]
    grads = torch.autograd.grad(out, [state[key] for key in _scan_inputs(state)], state["dy"])
    return [out.detach(), final.detach(), *grads]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ------------------------------------------------------------------------------- work


def work(case):
    size, op = _SIZE[case["dtype"]], case["op"]
    if op.startswith("norm"):
        rows, dim = case["rows"], case["dim"]
        two = 2 if case["residual"] else 1
        moved = size * (2 * two * rows * dim + dim)   # x, residual; y, total; the weight
        if op == "norm_8bit":
            moved -= (size - 1) * rows * dim - 4 * rows * (dim // (case["group"] or dim))
        if op == "norm_train":                        # dy, dtotal; dx, dresidual; dweight
            moved += size * (2 * two * rows * dim + dim)
        return {"bytes": moved, "flops": {"norm": 5, "norm_8bit": 8, "norm_train": 16}[op]
                * rows * dim}
    batch, dim = case["batch"], case["dim"]
    if op == "conv_step":
        width = case["width"]
        return {"bytes": size * dim * (batch * (2 + 2 * (width - 1)) + width + 1),
                "flops": batch * dim * (2 * width + 4)}
    # ragged lengths: the first full, the last of several empty, the others half on average;
    # outputs are whole (zeros after a sequence's end)
    full = batch if not case.get("ragged") else (1 if batch == 1 else 1 + (batch - 2) / 2)
    if op.startswith("conv"):
        width, length = case["width"], case["length"]
        read, written = int(full * length) * dim, batch * length * dim
        state = batch * (width - 1) * dim
        moved = read + written + state * (2 if case["initial"] else 1) + dim * (width + 1)
        flops = read * (2 * width + 4)
        if op == "conv_train":
            moved += read + written + dim * (width + 1)
            flops += read * (4 * width + 8)
        return {"bytes": size * moved, "flops": flops}
    states, groups = case["states"], case["groups"]
    token = (4 if case["gate"] else 3) * dim + 2 * groups * states   # x, dt, gate, b, c, and y
    params = 4 * dim * (states + 2)
    state = 4 * batch * dim * states
    if op == "scan_step":
        return {"bytes": size * batch * token + params + 2 * state,
                "flops": batch * dim * (7 * states + 12)}
    length = case["length"]
    read, written = int(full * length), batch * length
    moved = (size * (read * (token - dim) + written * dim) + params
             + state * (2 if case["initial"] else 1))
    flops = read * dim * (7 * states + 12)
    if op == "scan_train":   # dy; the gradients of everything read
        moved += size * (read * dim + written * (token - dim)) + params
        moved += state if case["initial"] else 0
        flops += read * dim * (16 * states + 24)
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------- definitions


def _exact_norm(state, case):
    x, w = state["x"].detach(), state["weight"].detach().double()
    total, outputs = x.double(), []
    if state["residual"] is not None:
        total = total + state["residual"].detach().double()
        outputs = [total]
    t = total.to(x.dtype).double()  # the norm is that of the sum as it is stored
    dim = t.shape[1]
    sigma = torch.sqrt((t * t).sum(1, keepdim=True) / dim + _EPS)
    y = t / sigma * w
    if case["op"] == "norm":
        return [y, *outputs]
    if case["op"] == "norm_8bit":
        cut = y.view(y.shape[0], -1, case["group"] or dim)
        scale = torch.linalg.vector_norm(cut, float("inf"), dim=2) / 448
        scale[scale == 0] = 1
        return [(cut / scale.unsqueeze(2)).view_as(y), scale, *outputs]
    dy = state["dy"].double()
    g = dy * w
    # through y = t w / sigma(t): direct, and through sigma
    dx = g / sigma - t * (g * t).sum(1, keepdim=True) / (dim * sigma ** 3)
    if state["dtotal"] is not None:
        dx = dx + state["dtotal"].double()
    return [y, *outputs, dx, *([dx] if outputs else []), (dy * t / sigma).sum(0)]


def _lengths(state, batch, length, device):
    n = state["lengths"]
    return torch.full((batch,), length, device=device) if n is None else n.long()


def _exact_conv(state, case):
    """Tap by tap over a padded copy of the tokens."""
    x, w, bias = (state[key].detach().double() for key in ("x", "weight", "bias"))
    batch, length, dim = x.shape
    width = case["width"]
    n = _lengths(state, batch, length, x.device)
    live = (torch.arange(length, device=x.device).view(1, -1) < n.view(-1, 1)).unsqueeze(2)
    line = torch.zeros(batch, length + width - 1, dim, device=x.device, dtype=torch.float64)
    line[:, width - 1:] = x.masked_fill(~live, 0)
    if state["initial"] is not None:
        line[:, :width - 1] = state["initial"].double()
    p = torch.zeros_like(x) + bias
    for j in range(width):
        p += w[:, j] * line[:, j:j + length]
    s = torch.sigmoid(p)
    y = (p * s if case["silu"] else p).masked_fill(~live, 0)
    final = torch.stack([line[i, n[i]:n[i] + width - 1] for i in range(batch)])
    if case["op"] == "conv":
        return [y, final]
    dp = state["dy"].double()
    if case["silu"]:
        dp = dp * (s + p * s * (1 - s))
    dp = dp.masked_fill(~live, 0)
    dline, dw = torch.zeros_like(line), torch.empty_like(w)
    for j in range(width):
        dline[:, j:j + length] += w[:, j] * dp
        dw[:, j] = (dp * line[:, j:j + length]).sum((0, 1))
    dx = dline[:, width - 1:].masked_fill(~live, 0)
    return [y, final, dx, dw, dp.sum((0, 1))]


def _exact_conv_step(state):
    pool = state["state"].double()
    w, bias = state["weight"].double(), state["bias"].double()
    rows = range(len(state["x"])) if state["slots"] is None else state["slots"].tolist()
    out = []
    for i, row in enumerate(rows):
        window = torch.cat([pool[row], state["x"][i:i + 1].double()])
        pool[row] = window[1:]
        p = torch.einsum("wd,dw->d", window, w) + bias
        out.append(p * torch.sigmoid(p))
    return [torch.stack(out), pool]


def _exact_scan(state, case):
    """The recurrence token by token; for gradients the adjoint recurrence back in time."""
    x, dt, a, b, c, skip = (state[key].detach().double()
                            for key in ("x", "dt", "a", "b", "c", "skip"))
    batch, length, dim = x.shape
    groups, states = case["groups"], case["states"]
    v = dt + state["dt_bias"].detach().double()
    n = _lengths(state, batch, length, x.device)
    live = torch.arange(length, device=x.device).view(1, -1) < n.view(-1, 1)
    delta = torch.logaddexp(v, torch.zeros_like(v)).masked_fill(~live.unsqueeze(2), 0)
    x = x.masked_fill(~live.unsqueeze(2), 0)
    b, c = (t.masked_fill(~live.view(batch, length, 1, 1), 0) for t in (b, c))
    gate = None
    opened = torch.ones_like(x)
    if state["gate"] is not None:
        gate = state["gate"].detach().double().masked_fill(~live.unsqueeze(2), 0)
        opened = gate * torch.sigmoid(gate)
    # channels by group: (B, G, D / G, N)
    per = dim // groups
    shape = (batch, groups, per, states)
    a4 = a.view(1, groups, per, states)
    h = torch.zeros(shape, device=x.device, dtype=torch.float64)
    if state["initial"] is not None:
        h = state["initial"].detach().double().view(shape).clone()
    train = case["op"] == "scan_train"
    kept = [h.clone()] if train else []
    y = torch.empty(length, batch, groups, per, device=x.device, dtype=torch.float64)
    d5, u5 = (t.view(batch, length, groups, per, 1) for t in (delta, delta * x))
    for t in range(length):
        h.mul_(torch.exp(d5[:, t] * a4)).addcmul_(u5[:, t], b[:, t].unsqueeze(2))
        torch.matmul(h, c[:, t].unsqueeze(3), out=y[t].unsqueeze_(3))
        if train:
            kept.append(h.clone())
    p = y.view(length, batch, dim).transpose(0, 1) + skip * x
    result = [p * opened, h.view(batch, dim, states)]
    if not train:
        return result

    dy = state["dy"].double().masked_fill(~live.unsqueeze(2), 0)
    dp = dy * opened
    q5 = dp.view(batch, length, groups, per, 1)
    g = torch.zeros_like(h)
    da = torch.zeros_like(a4)
    dx, ddelta = torch.empty_like(x), torch.empty_like(x)
    db, dc = torch.empty_like(b), torch.empty_like(c)
    for t in range(length - 1, -1, -1):
        g.addcmul_(q5[:, t], c[:, t].unsqueeze(2))
        dc[:, t] = (q5[:, t] * kept[t + 1]).sum(2)
        db[:, t] = (u5[:, t] * g).sum(2)
        into = (g * b[:, t].unsqueeze(2)).sum(3).view(batch, dim)
        dx[:, t] = into * delta[:, t]
        g.mul_(torch.exp(d5[:, t] * a4))
        by_rate = g * kept[t]
        ddelta[:, t] = (by_rate * a4).sum(3).view(batch, dim) + into * x[:, t]
        da += (by_rate * d5[:, t]).sum(0, keepdim=True)
    ddt = ddelta * torch.sigmoid(v)
    ddt = ddt.masked_fill(~live.unsqueeze(2), 0)
    grads = {"x": dx + skip * dp, "dt": ddt, "a": da.view(dim, states), "b": db, "c": dc,
             "skip": (dp * x).sum((0, 1)), "dt_bias": ddt.sum((0, 1)),
             "initial": g.view(batch, dim, states)}
    if gate is not None:
        s = torch.sigmoid(gate)
        grads["gate"] = dy * p * (s + gate * s * (1 - s))
    return result + [grads[key] for key in _scan_inputs(state)]


def _exact_scan_step(state):
    pool, a = state["state"].double(), state["a"].double()
    dim = a.shape[0]
    v = state["dt"].double() + state["dt_bias"].double()
    delta = torch.logaddexp(v, torch.zeros_like(v))
    x, b, c, gate = (state[key].double() for key in ("x", "b", "c", "gate"))
    of = torch.arange(dim, device=a.device) // (dim // b.shape[1])
    rows = range(len(x)) if state["slots"] is None else state["slots"].tolist()
    out = []
    for i, row in enumerate(rows):
        h = torch.exp(delta[i].unsqueeze(1) * a) * pool[row]
        h = h + (delta[i] * x[i]).unsqueeze(1) * b[i, of]
        pool[row] = h
        p = torch.einsum("dn,dn->d", h, c[i, of]) + state["skip"].double() * x[i]
        out.append(p * gate[i] * torch.sigmoid(gate[i]))
    return [torch.stack(out), pool]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op.startswith("norm"):
            return _exact_norm(state, case)
        if op == "conv_step":
            return _exact_conv_step(state)
        if op == "scan_step":
            return _exact_scan_step(state)
        return _exact_conv(state, case) if op.startswith("conv") else _exact_scan(state, case)
