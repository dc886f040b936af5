"""What is measured of the token-model operators: layer norm, linear attention with a decay for
each head, and its single-token form.

Every case is a dict of plain values; ``op`` says which operator it calls:

* ``norm``        ``layer_norm`` of ``(rows, dim)``
* ``norm_train``  the same with its gradients (input, weight, bias)
* ``prompt``      ``linear_attention`` over whole sequences, with the state after them
* ``train``       the same with its gradients (queries, keys, values)
* ``step``        ``linear_attention_step``: one token for every sequence, states updated in place

``run`` computes a case in elementary torch operations in 32 bits, or, with ``own`` set, through
the package's public functions.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------- the cases


def _norm(op, rows, dim, dtype):
    return {"op": op, "rows": rows, "dim": dim, "dtype": dtype}


def _mix(op, batch, length, heads, kv_heads, dk, dv, dtype, ragged=False, initial=False):
    return {"op": op, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads,
            "dk": dk, "dv": dv, "dtype": dtype, "ragged": ragged, "initial": initial}


def _step(batch, heads, kv_heads, dk, dv, dtype, pool):
    return {"op": "step", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dk": dk,
            "dv": dv, "dtype": dtype, "pool": pool}


def listed():
    cases = {
        # the norm before one decoded token of a few sequences: latency
        "norm_tokens": _norm("norm", 4, 256, "bf16"),
        # a long batch of signals' tokens at an odd width, inference
        "norm_odd_f32": _norm("norm", 40000, 1001, "f32"),
        # a training batch of the token mixers' width (8 x 4096 tokens of 256)
        "norm_train_mixer_f16": _norm("norm_train", 8 * 4096, 256, "f16"),
        # a large training batch of a wide model
        "norm_train_large": _norm("norm_train", 65536, 2048, "bf16"),
        # a short question: latency
        "prompt_short": _mix("prompt", 1, 37, 4, 4, 64, 64, "bf16"),
        # the token mixers' shape (8, 4096, 256), four heads
        "prompt_mixer": _mix("prompt", 8, 4096, 4, 4, 64, 64, "bf16"),
        # prompts of different lengths (an empty one among them) continued from states, shared
        # heads, uneven head sizes, full precision
        "prompt_ragged_f32": _mix("prompt", 5, 1537, 6, 2, 48, 80, "f32", True, True),
        # one long document
        "prompt_long": _mix("prompt", 1, 65536, 16, 16, 128, 128, "bf16"),
        # a training step's attention
        "train_wide": _mix("train", 4, 4096, 16, 16, 64, 64, "bf16"),
        # the same with shared heads, continued from states, at an odd length
        "train_shared_f16": _mix("train", 3, 2501, 8, 4, 128, 128, "f16", False, True),
        # one token of one sequence: latency
        "step_one": _step(1, 4, 4, 64, 64, "bf16", 0),
        # one token for each of a full pool of sequences
        "step_pool": _step(240, 16, 16, 128, 128, "bf16", 256),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "norm_train", "prompt", "prompt", "train", "train", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "norm_train"):
        dim = _log_int(rng, 16, 8192)
        if rng.random() < 0.5:
            dim = max(16, dim // 64 * 64)
        most = 2 ** (28 if op == "norm" else 26) // _SIZE[dtype] // dim
        return _norm(op, _log_int(rng, 1, max(1, min(65536, most))), dim, dtype)
    heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    kv_heads = rng.choice([g for g in range(1, heads + 1) if heads % g == 0])
    sizes = [16, 32, 40, 48, 64, 64, 64, 80, 96, 128, 128, 128]
    dk = rng.choice(sizes)
    dv = dk if rng.random() < 0.7 else rng.choice(sizes)
    if op == "step":
        batch = _log_int(rng, 1, 240)
        return _step(batch, heads, kv_heads, dk, dv, dtype,
                     0 if rng.random() < 0.5 else batch + rng.randrange(1, 17))
    tokens = 65536 if op == "prompt" else 16384
    batch = _log_int(rng, 1, 16)
    length = _log_int(rng, 1, (tokens if dtype != "f32" else tokens // 4) // batch)
    return _mix(op, batch, length, heads, kv_heads, dk, dv, dtype, rng.random() < 0.4,
                rng.random() < 0.4)


# ------------------------------------------------------------------------------- inputs


def _schedule(heads, device):
    """Log decays spread over the heads, from about 1/32 to 1/4096 lost a token."""
    rate = [2.0 ** -(5 + 7 * h / max(1, heads - 1)) for h in range(heads)]
    return torch.tensor([math.log1p(-r) for r in rate], dtype=torch.float32, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device=device) * scale).to(to)

    state = {"case": case}
    if case["op"] in ("norm", "norm_train"):
        rows, dim = case["rows"], case["dim"]
        # activations with a mean and a few strong channels, as residual streams have
        x = torch.randn(rows, dim, generator=gen, device=device)
        x += torch.randn(dim, generator=gen, device=device)
        state["x"] = x.to(dtype)
        state["weight"] = (1 + 0.1 * torch.randn(dim, generator=gen, device=device)).to(dtype)
        state["bias"] = normal(dim, scale=0.1)
        if case["op"] == "norm_train":
            state["dy"] = normal(rows, dim)
            for key in ("x", "weight", "bias"):
                state[key].requires_grad_()
        return state

    b, h, hk, dk, dv = (case[key] for key in ("batch", "heads", "kv_heads", "dk", "dv"))
    state["log_decay"] = _schedule(h, device)
    if case["op"] == "step":
        state["q"], state["k"] = normal(b, h, dk), normal(b, hk, dk)
        state["v"] = normal(b, hk, dv)
        pool = case["pool"]
        state["state"] = normal(pool or b, h, dk, dv, scale=4.0, to=torch.float32)
        state["slots"] = None
        if pool:
            order = torch.randperm(pool, generator=gen, device=device)
            state["slots"] = order[:b].to(torch.int32)
        return state

    length = case["length"]
    state["q"] = normal(b, length, h, dk)
    state["k"] = normal(b, length, hk, dk)
    state["v"] = normal(b, length, hk, dv)
    state["initial"] = None
    if case["initial"]:
        state["initial"] = normal(b, h, dk, dv, scale=4.0, to=torch.float32)
    state["lengths"] = None
    if case["ragged"]:
        lengths = torch.randint(0, length + 1, (b,), generator=gen, device=device)
        lengths[0] = length
        if b > 1:
            lengths[-1] = 0
        state["lengths"] = lengths.to(torch.int32)
    if case["op"] == "train":
        state["do"] = normal(b, length, h, dv)
        for key in ("q", "k", "v"):
            state[key].requires_grad_()
    return state


# ------------------------------------------------------------------------------- plain forms


def _plain_norm(x, weight, bias, eps=1e-5):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = (centred.square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = centred * rstd
    return hat * weight.float() + bias.float(), hat, rstd


def _plain_norm_train(x, weight, bias, dy):
    y, hat, rstd = _plain_norm(x, weight, bias)
    dy = dy.float()
    g = dy * weight.float()
    dx = rstd * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    return y, dx, (dy * hat).sum(0), dy.sum(0)


def _chunks(x, n, size):
    """(B, L, H, D) -> (B, H, n, size, D), zeros after the last token."""
    b, length, h, d = x.shape
    padded = x.new_zeros(b, n * size, h, d)
    padded[:, :length] = x
    return padded.view(b, n, size, h, d).permute(0, 3, 1, 2, 4)


def _plain_mix(q, k, v, log_decay, start):
    """Unscaled linear attention of fp32 (B, L, H, D) from the state ``start``, in chunks."""
    b, length, h, dk = q.shape
    dv = v.shape[-1]
    size = 128
    n = (length + size - 1) // size
    qc, kc, vc = (_chunks(x, n, size) for x in (q, k, v))
    step = torch.arange(size, device=q.device, dtype=torch.float32)
    a = log_decay.view(1, h, 1, 1, 1)
    gap = step.view(-1, 1) - step
    mask = torch.exp(a * gap.clamp(min=0)) * (gap >= 0)
    out = torch.matmul(torch.matmul(qc, kc.transpose(-1, -2)) * mask, vc)
    read = torch.exp(a * (step + 1).view(-1, 1))
    write = torch.exp(a * (size - 1 - step).view(-1, 1))
    update = torch.matmul((kc * write).transpose(-1, -2), vc)
    states = torch.empty(b, h, n, dk, dv, device=q.device)
    whole = torch.exp(log_decay * size).view(1, h, 1, 1)
    current = start
    for i in range(n):
        states[:, :, i] = current
        current = whole * current + update[:, :, i]
    out = out + torch.matmul(qc * read, states)
    return out.permute(0, 2, 3, 1, 4).reshape(b, n * size, h, dv)[:, :length]


def _shared(x, heads):
    """Keys or values repeated for the heads that share them, in 32 bits."""
    return x.float().repeat_interleave(heads // x.shape[2], dim=2)


def _valid(state, length):
    lengths = state["lengths"]
    if lengths is None:
        return None
    t = torch.arange(length, device=lengths.device)
    return (t.view(1, -1) < lengths.view(-1, 1)).view(-1, length, 1, 1)


def _plain_sequence(state, q, k, v, with_state):
    """Outputs (scaled) and the state after the last valid token, fp32."""
    b, length, h, dk = q.shape
    scale = dk ** -0.5
    valid = _valid(state, length)
    if valid is not None:
        k, v = torch.where(valid, k, 0.0), torch.where(valid, v, 0.0)
    a = state["log_decay"]
    start = state["initial"]
    if start is None:
        start = torch.zeros(b, h, dk, v.shape[-1], device=q.device)
    out = scale * _plain_mix(q, k, v, a, start)
    if valid is not None:
        out = torch.where(valid, out, 0.0)
    if not with_state:
        return out, None
    n = state["lengths"]
    n = torch.full((b,), length, device=q.device) if n is None else n
    age = (n.view(b, 1) - 1 - torch.arange(length, device=q.device).view(1, length))
    weight = torch.exp(a.view(1, 1, h) * age.clamp(min=0).unsqueeze(-1))
    final = torch.matmul((k * weight.unsqueeze(-1)).permute(0, 2, 3, 1), v.permute(0, 2, 1, 3))
    final = final + torch.exp(a.view(1, h) * n.view(b, 1)).view(b, h, 1, 1) * start
    return out, final


def _plain_train(state):
    q, k, v, do = (state[key].detach() for key in ("q", "k", "v", "do"))
    dtype = q.dtype
    b, length, h, dk = q.shape
    hk, dv = v.shape[2], v.shape[3]
    scale = dk ** -0.5
    q, do, k, v = q.float(), do.float(), _shared(k, h), _shared(v, h)
    out, final = _plain_sequence(state, q, k, v, True)
    valid = _valid(state, length)
    if valid is not None:
        q, k, v, do = (torch.where(valid, x, 0.0) for x in (q, k, v, do))
    a = state["log_decay"]
    start = state["initial"]
    if start is None:
        start = torch.zeros(b, h, dk, dv, device=q.device)
    # each gradient is the operator again, with other operands or in reversed time
    dq = scale * _plain_mix(do, v, k, a, start.transpose(-1, -2))
    none = torch.zeros_like(start)
    rev = [x.flip(1) for x in (q, k, v, do)]
    grad_v = scale * _plain_mix(rev[1], rev[0], rev[3], a, none).flip(1)
    grad_k = scale * _plain_mix(rev[2], rev[3], rev[0], a, none.transpose(-1, -2)).flip(1)
    if valid is not None:
        dq, grad_k, grad_v = (torch.where(valid, x, 0.0) for x in (dq, grad_k, grad_v))
    grad_k = grad_k.reshape(b, length, hk, h // hk, dk).sum(3)
    grad_v = grad_v.reshape(b, length, hk, h // hk, dv).sum(3)
    return [out.to(dtype), final, dq.to(dtype), grad_k.to(dtype), grad_v.to(dtype)]


def _plain_step(state):
    q, k, v = state["q"].float(), state["k"].float(), state["v"].float()
    h = q.shape[1]
    group = h // k.shape[1]
    k, v = k.repeat_interleave(group, dim=1), v.repeat_interleave(group, dim=1)
    pool, slots = state["state"], state["slots"]
    current = pool if slots is None else pool[slots.long()]
    decay = torch.exp(state["log_decay"]).view(1, h, 1, 1)
    current = decay * current + k.unsqueeze(-1) * v.unsqueeze(-2)
    out = q.shape[-1] ** -0.5 * (q.unsqueeze(-1) * current).sum(-2)
    if slots is None:
        pool.copy_(current)
    else:
        pool[slots.long()] = current
    return [out.to(state["q"].dtype), pool]


def _run_plain(state):
    op = state["case"]["op"]
    if op == "norm":
        x = state["x"]
        return _plain_norm(x, state["weight"], state["bias"])[0].to(x.dtype)
    if op == "norm_train":
        x = state["x"].detach()
        grads = _plain_norm_train(x, state["weight"].detach(), state["bias"].detach(),
                                  state["dy"])
        return [g.to(x.dtype) for g in grads]
    if op == "prompt":
        h, dtype = state["q"].shape[2], state["q"].dtype
        out, final = _plain_sequence(state, state["q"].float(), _shared(state["k"], h),
                                     _shared(state["v"], h), True)
        return [out.to(dtype), final]
    if op == "train":
        return _plain_train(state)
    return _plain_step(state)


# ------------------------------------------------------------------------------- own kernels


def _run_own(state):
    import pytorch_morlet_fdwt_b200 as fdwt

    op = state["case"]["op"]
    if op == "norm":
        return fdwt.layer_norm(state["x"], state["weight"], state["bias"])
    if op == "norm_train":
        inputs = (state["x"], state["weight"], state["bias"])
        y = fdwt.layer_norm(*inputs)
        return [y.detach(), *torch.autograd.grad(y, inputs, state["dy"])]
    if op in ("prompt", "train"):
        out, final = fdwt.linear_attention(state["q"], state["k"], state["v"],
                                           state["log_decay"], initial_state=state["initial"],
                                           lengths=state["lengths"])
        if op == "prompt":
            return [out, final]
        grads = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"])
        return [out.detach(), final.detach(), *grads]
    out = fdwt.linear_attention_step(state["q"], state["k"], state["v"], state["log_decay"],
                                     state["state"], slots=state["slots"])
    return [out, state["state"]]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ------------------------------------------------------------------------------- work


def work(case):
    size = _SIZE[case["dtype"]]
    op = case["op"]
    if op in ("norm", "norm_train"):
        rows, dim = case["rows"], case["dim"]
        moves = 2 if op == "norm" else 4    # x, y; and dy, dx
        params = 2 if op == "norm" else 4   # weight, bias; and their gradients
        return {"bytes": size * (moves * rows * dim + params * dim),
                "flops": (8 if op == "norm" else 22) * rows * dim}
    b, h, hk, dk, dv = (case[key] for key in ("batch", "heads", "kv_heads", "dk", "dv"))
    if op == "step":
        token = size * (h * dk + hk * (dk + dv) + h * dv)
        return {"bytes": b * (token + 8 * h * dk * dv), "flops": 5 * b * h * dk * dv}
    length = case["length"]
    state = 4 * b * h * dk * dv
    # ragged lengths: the first full, the last of several empty, the others half on average;
    # outputs are whole (zeros after a sequence's end)
    full = b if not case["ragged"] else (1 if b == 1 else 1 + (b - 2) / 2)
    read, written = int(full * length), b * length
    q, kv, o = h * dk, hk * (dk + dv), h * dv
    moved = size * (read * (q + kv) + written * o) + state * (2 if case["initial"] else 1)
    flops = 4 * read * h * dk * dv
    if op == "train":  # do read, dq, dk and dv written
        moved += size * (read * o + written * (q + kv))
        flops += 10 * read * h * dk * dv
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------------------- definitions


def _exact_norm(state, case):
    x = state["x"].detach().double()
    w, c = state["weight"].detach().double(), state["bias"].detach().double()
    dim = x.shape[1]
    mean = x.sum(1, keepdim=True) / dim
    var = (x * x).sum(1, keepdim=True) / dim - mean * mean
    sigma = torch.sqrt(var + 1e-5)
    y = (x - mean) / sigma * w + c
    if case["op"] == "norm":
        return y
    dy = state["dy"].double()
    g = dy * w
    # dL/dx through y = (x - mean) / sigma: direct, through the mean, through the variance
    through_var = (g * (x - mean)).sum(1, keepdim=True) / (dim * sigma ** 3)
    dx = g / sigma - g.sum(1, keepdim=True) / (dim * sigma) - (x - mean) * through_var
    return [y, dx, (dy * (x - mean) / sigma).sum(0), dy.sum(0)]


def _exact_recurrence(state, case):
    """The recurrence token by token, S = d S + k v^T, o = scale q S; for gradients the adjoint
    recurrence back in time."""
    q, k, v = (state[key].detach().double() for key in ("q", "k", "v"))
    b, length, h, dk = q.shape
    hk, dv = v.shape[2], v.shape[3]
    train = case["op"] == "train"
    head = torch.arange(h, device=q.device) // (h // hk)
    k, v = k[:, :, head], v[:, :, head]
    decay = torch.exp(state["log_decay"].double())
    scale = 1.0 / math.sqrt(dk)
    lengths = state["lengths"]
    if lengths is None:
        lengths = torch.full((b,), length, device=q.device)
    t = torch.arange(length, device=q.device)
    live = (t.view(-1, 1) < lengths.view(1, -1)).repeat_interleave(h, dim=1)  # (L, B*H)
    keep = torch.where(live, decay.repeat(b), 1.0).view(length, b * h, 1, 1)
    live = live.to(torch.float64).unsqueeze(-1)

    def rows(x):  # (L, B*H, D), zero after the sequence's end
        return x.permute(1, 0, 2, 3).reshape(length, b * h, -1) * live

    q, k, v = rows(q), rows(k), rows(v)
    s = torch.zeros(b * h, dk, dv, device=q.device, dtype=torch.float64)
    if state["initial"] is not None:
        s = state["initial"].double().reshape(b * h, dk, dv).clone()
    out = torch.empty(length, b * h, 1, dv, device=q.device, dtype=torch.float64)
    if train:
        do = rows(state["do"].double())
        dq = torch.empty(length, b * h, dk, 1, device=q.device, dtype=torch.float64)
    for i in range(length):
        s.mul_(keep[i]).baddbmm_(k[i].unsqueeze(2), v[i].unsqueeze(1))
        torch.bmm(q[i].unsqueeze(1), s, out=out[i])
        if train:
            torch.bmm(s, do[i].unsqueeze(2), out=dq[i])

    def tokens(x, heads_of=None):
        x = x.reshape(length, b, h, -1).permute(1, 0, 2, 3)
        if heads_of is None:
            return x
        return x.reshape(b, length, heads_of, h // heads_of, -1).sum(3)

    result = [tokens(out * scale * live.unsqueeze(-1)), s.reshape(b, h, dk, dv)]
    if not train:
        return result
    r = torch.zeros_like(s)
    grad_k, grad_v = torch.empty_like(dq), torch.empty_like(out)
    for i in range(length - 1, -1, -1):
        r.baddbmm_(q[i].unsqueeze(2), do[i].unsqueeze(1))
        torch.bmm(r, v[i].unsqueeze(2), out=grad_k[i])
        torch.bmm(k[i].unsqueeze(1), r, out=grad_v[i])
        r.mul_(keep[i])
    return result + [tokens(dq * scale), tokens(grad_k * scale, hk), tokens(grad_v * scale, hk)]


def _exact_step(state):
    q, k, v = (state[key].double() for key in ("q", "k", "v"))
    b, h, dk = q.shape
    head = torch.arange(h, device=q.device) // (h // k.shape[1])
    pool = state["state"].double()
    slots = range(b) if state["slots"] is None else state["slots"].tolist()
    decay = torch.exp(state["log_decay"].double())
    out = []
    for i, slot in enumerate(slots):
        s = decay.view(h, 1, 1) * pool[slot] + torch.einsum("hk,hv->hkv", k[i, head], v[i, head])
        pool[slot] = s
        out.append(torch.einsum("hk,hkv->hv", q[i], s) / math.sqrt(dk))
    return [torch.stack(out), pool]


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("norm", "norm_train"):
            return _exact_norm(state, case)
        if case["op"] == "step":
            return _exact_step(state)
        return _exact_recurrence(state, case)
