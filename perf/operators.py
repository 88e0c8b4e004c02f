"""Measured cases of the operators around the training step: the gated feed-forward
product, rotary positions, and the global gradient norm with clipping.

``listed()`` and ``draw()`` give cases, ``prepare()`` what a program holds before the
call, ``run()`` one call (in elementary torch operations, or through ``scao_b200`` where
``own`` is true), ``work()`` what it has to move and compute, ``exact()`` its value in
64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a 2048 x 8192 block: both weight matrices are read once
        {"name": "ff_token", "op": "ff", "rows": 1, "d": 2048, "ff": 8192, "act": "silu",
         "dtype": "bf16", "train": False},
        # a short batch of rows at GPT-2-medium width, the tanh form of GELU
        {"name": "ff_batch", "op": "ff", "rows": 40, "d": 1024, "ff": 4096, "act": "gelu_tanh",
         "dtype": "fp16", "train": False},
        # the training step of a test-sized model (8 x 64 tokens): latency
        {"name": "ff_small_train", "op": "ff", "rows": 512, "d": 128, "ff": 512, "act": "silu",
         "dtype": "bf16", "train": True},
        # evaluation over a GPT-2-medium batch (8 x 1024 tokens)
        {"name": "ff_eval", "op": "ff", "rows": 8192, "d": 1024, "ff": 4096, "act": "silu",
         "dtype": "bf16", "train": False},
        # training at the Llama-1B layer's shape (2 x 2048 tokens): the largest
        {"name": "ff_train", "op": "ff", "rows": 4096, "d": 2048, "ff": 8192, "act": "silu",
         "dtype": "bf16", "train": True},
        # training with sizes that divide by nothing: a packed batch, an odd inner width
        {"name": "ff_train_odd", "op": "ff", "rows": 1531, "d": 1000, "ff": 2731, "act": "gelu",
         "dtype": "fp16", "train": True},
        # one new token for each of 32 sequences, far into them, grouped heads
        {"name": "rope_token", "op": "rope", "batch": 32, "len": 1, "heads": 32, "kv": 8,
         "head_dim": 64, "dim": 64, "interleaved": False, "scaling": "none", "start": 130000,
         "dtype": "bf16", "train": False},
        # the attention input of a GPT-2-medium batch, views of the fused projection
        {"name": "rope_train", "op": "rope", "batch": 8, "len": 1024, "heads": 16, "kv": 16,
         "head_dim": 64, "dim": 64, "interleaved": False, "scaling": "none", "start": 0,
         "dtype": "bf16", "train": True},
        # one long sequence scaled beyond its training length, part of the head, interleaved
        {"name": "rope_long", "op": "rope", "batch": 1, "len": 30011, "heads": 12, "kv": 2,
         "head_dim": 80, "dim": 64, "interleaved": True, "scaling": "yarn", "start": 100000,
         "dtype": "fp32", "train": False},
        # the gradients of a test-sized model: latency
        {"name": "clip_small", "op": "clip", "layers": 2, "d": 128, "ff": 512, "vocab": 512,
         "dtype": "fp32", "norm": "2", "max_norm": 1.0, "aligned": True},
        # GPT-2-medium, fp32 gradients (355 M values), clipped
        {"name": "clip_medium", "op": "clip", "layers": 24, "d": 1024, "ff": 4096, "vocab": 50257,
         "dtype": "fp32", "norm": "2", "max_norm": 1.0, "aligned": True},
        # fp32, bf16 and fp16 gradients of odd sizes packed without alignment, largest value
        {"name": "clip_mixed", "op": "clip", "layers": 6, "d": 771, "ff": 2049, "vocab": 32003,
         "dtype": "mixed", "norm": "inf", "max_norm": 1e-3, "aligned": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ff", "rope", "clip"])
    if op == "ff":
        step = rng.choice([1, 2, 8, 64])
        size = lambda lo, hi: max(step, _log(rng, lo, hi) // step * step)  # noqa: E731
        return {"op": op, "rows": _log(rng, 1, 4096), "d": size(64, 2048), "ff": size(64, 8192),
                "act": rng.choice(["silu", "gelu", "gelu_tanh"]), "dtype": rng.choice(["bf16", "fp16"]),
                "train": rng.random() < 0.5}
    if op == "rope":
        head_dim = rng.choice([32, 64, 80, 96, 100, 128, 256])
        dim = head_dim if rng.random() < 0.5 else rng.randrange(2, head_dim + 1, 2)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        total = _log(rng, 1, 32000000 // ((heads + kv) * head_dim))
        batch = min(total, _log(rng, 1, 64))
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"op": op, "batch": batch, "len": max(1, total // batch), "heads": heads, "kv": kv,
                "head_dim": head_dim, "dim": dim, "interleaved": rng.random() < 0.5,
                "scaling": "none" if scaling == "ntk" and dim == 2 else scaling,
                "start": rng.choice([0, _log(rng, 1, 1000000)]),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "train": rng.random() < 0.5}
    layers, d = _log(rng, 1, 32), _log(rng, 16, 1024)
    return {"op": op, "layers": layers, "d": d, "ff": _log(rng, d, 4 * d),
            "vocab": _log(rng, 64, 50000) if layers < 24 else 64,
            "dtype": rng.choice(["fp32", "bf16", "fp16", "mixed"]), "norm": rng.choice(["2", "inf", "1"]),
            "max_norm": rng.choice([1e-3, 1.0, 1e9]), "aligned": rng.random() < 0.5}


# --------------------------------------------------------------------------- inputs
def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _grad_sizes(c):
    """(elements, dtype) of every gradient: embedding, then per layer the two norms with
    their biases, the fused projection, the output and the two feed-forward matrices."""
    d, ff = c["d"], c["ff"]
    sizes = [c["vocab"] * d] + [n for _ in range(c["layers"])
                                for n in (d, d, 3 * d * d, d * d, d, d, ff * d, d * ff)] + [d, d]
    cycle = ["fp32", "bf16", "fp16"] if c["dtype"] == "mixed" else [c["dtype"]]
    return [(n, cycle[i % len(cycle)]) for i, n in enumerate(sizes)]


def _scale(i):
    """The standard deviation of gradient ``i``."""
    return 1e-3 * 2.0 ** (i % 5)


def _expected_norm(c):
    """About the norm of ``_prepare_clip``'s gradients; a fifth of the embedding's rows is set."""
    each = [(n * 0.2 if i == 0 else n, _scale(i)) for i, (n, _) in enumerate(_grad_sizes(c))]
    if c["norm"] == "inf":
        return max(s * math.sqrt(2 * math.log(n + 2)) for n, s in each)
    if c["norm"] == "1":
        return sum(n * s for n, s in each) * math.sqrt(2 / math.pi)
    return math.sqrt(sum(n * s * s for n, s in each))


def _prepare_clip(c, gen):
    sizes = _grad_sizes(c)
    flats, params = {}, []
    pitch = lambda n: -(-n // 64) * 64 if c["aligned"] else n  # noqa: E731
    for kind in sorted({k for _, k in sizes}):
        flats[kind] = torch.zeros(sum(pitch(n) for n, k in sizes if k == kind),
                                  dtype=DTYPES[kind], device="cuda")
    at = dict.fromkeys(flats, 0)
    for i, (n, kind) in enumerate(sizes):
        grad = flats[kind][at[kind]:at[kind] + n]
        at[kind] += pitch(n)
        scale = _scale(i)
        if i == 0:      # an embedding's gradient: most rows saw no token
            rows = torch.rand(c["vocab"], generator=gen, device="cuda") < 0.2
            grad.view(c["vocab"], -1).copy_(_normal(gen, (c["vocab"], n // c["vocab"]), torch.float32, scale)
                                            * rows[:, None])
        else:
            grad.copy_(_normal(gen, (n,), torch.float32, scale))
        p = torch.nn.Parameter(torch.empty(n, dtype=DTYPES[kind], device="cuda"))
        p.grad = grad
        params.append(p)
    return {"params": params, "flats": [flats[k] for k in sorted(flats)], "max_norm": c["max_norm"]}


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": c}
    if c["op"] == "ff":
        t, m, d, f = DTYPES[c["dtype"]], c["rows"], c["d"], c["ff"]
        state.update(x=_normal(gen, (m, d), t), w_gate=_normal(gen, (f, d), t, d ** -0.5),
                     w_up=_normal(gen, (f, d), t, d ** -0.5))
        if c["train"]:
            state["dh"] = _normal(gen, (m, f), t, 0.1)
            for k in ("x", "w_gate", "w_up"):
                state[k].requires_grad_()
    elif c["op"] == "rope":
        t, b, n, h, kv, hd = (DTYPES[c["dtype"]], c["batch"], c["len"], c["heads"], c["kv"],
                              c["head_dim"])
        qkv = _normal(gen, (b, n, h + 2 * kv, hd), t)      # the fused projection's output
        state["q"], state["k"] = qkv[:, :, :h].transpose(1, 2), qkv[:, :, h:h + kv].transpose(1, 2)
        first = torch.randint(0, c["start"] + 1, (b, 1), generator=gen, device="cuda")
        state["positions"] = first + torch.arange(n, device="cuda")
        if c["train"]:
            for k in ("q", "k"):
                state[k] = state[k].detach().requires_grad_()
                state["d" + k] = _normal(gen, tuple(state[k].shape), t)
        if own:
            state["rotary"] = _rotary(c)
    else:
        state.update(_prepare_clip(c, gen))
    return state


# --------------------------------------------------------------------------- frequencies
SCALE, TRAINED, BASE, FAST, SLOW = 8.0, 8192, 10000.0, 32.0, 1.0


def _rotary(c):
    from scao_b200 import Rotary, RotaryScaling
    s = c["scaling"]
    scaling = None if s == "none" else RotaryScaling(s, SCALE, original_len=TRAINED)
    return Rotary(c["dim"], base=BASE, interleaved=c["interleaved"], scaling=scaling)


def _frequencies(c):
    """(radians per position in 64 bits, factor on the rotated values)."""
    dim = c["dim"]
    base = BASE * SCALE ** (dim / (dim - 2)) if c["scaling"] == "ntk" else BASE
    freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    if c["scaling"] == "linear":
        freq = freq / SCALE
    if c["scaling"] == "yarn":
        turns = TRAINED * freq / (2 * math.pi)
        keep = ((turns - SLOW) / (FAST - SLOW)).clamp(0, 1)
        return freq * keep + freq / SCALE * (1 - keep), 0.1 * math.log(SCALE) + 1
    return freq, 1.0


# --------------------------------------------------------------------------- plain forms
def _act(g, kind):
    """(activation, its derivative), by their definitions."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if kind == "gelu":
        phi = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    a, b = (2 / math.pi) ** 0.5, 0.044715
    t = torch.tanh(a * (g + b * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)


def _plain_ff(s):
    c, t = s["case"], s["x"].dtype
    x, wg, wu = (s[k].detach().float() for k in ("x", "w_gate", "w_up"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, c["act"])
    h = (a * u).to(t)
    if not c["train"]:
        return h
    dh = s["dh"].float()
    dg, du = dh * u * da, dh * a
    return [h] + [y.to(t) for y in (dg @ wg + du @ wu, dg.T @ x, du.T @ x)]


def _turn(x, cos, sin, interleaved):
    """The rotation of the first 2 * cos.shape[-1] values of each head."""
    n = cos.shape[-1]
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        out[..., :n], out[..., n:2 * n] = a * cos - b * sin, a * sin + b * cos
    return out


def _plain_rope(s):
    c = s["case"]
    freq, factor = _frequencies(c)
    angle = (s["positions"].double()[..., None] * freq)[:, None]
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    t = s["q"].dtype
    out = [_turn(s[k].detach().float(), cos, sin, c["interleaved"]).to(t) for k in ("q", "k")]
    if c["train"]:      # the rotation's transpose turns the gradient back
        out += [_turn(s[k].float(), cos, -sin, c["interleaved"]).to(t) for k in ("dq", "dk")]
    return out


def _plain_clip(s):
    c, grads = s["case"], [p.grad for p in s["params"]]
    if c["norm"] == "inf":
        total = torch.stack([g.abs().max().float() for g in grads]).max()
    elif c["norm"] == "1":
        total = torch.stack([g.float().abs().sum(dtype=torch.float64) for g in grads]).sum().float()
    else:
        total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt().float()
    coef = (s["max_norm"] / (total + 1e-6)).clamp(max=1.0)
    [g.copy_(g.float() * coef) for g in grads]
    return [total] + s["flats"]


def run(state):
    c = state["case"]
    if c["op"] == "clip":
        if own:
            from scao_b200 import clip_grad_norm_
            out = [clip_grad_norm_(state["params"], state["max_norm"], norm_type=float(c["norm"]))]
            out += state["flats"]
        else:
            out = _plain_clip(state)
        # the program's threshold decays slowly: a pass over the clipped gradients clips again
        state["max_norm"] *= 0.9999
        return out
    if not own:
        return _plain_ff(state) if c["op"] == "ff" else _plain_rope(state)
    if c["op"] == "ff":
        from scao_b200 import gated_ff
        h = gated_ff(state["x"], state["w_gate"], state["w_up"], activation=c["act"])
        if not c["train"]:
            return h
        return [h.detach(), *torch.autograd.grad(h, [state["x"], state["w_gate"], state["w_up"]], state["dh"])]
    q, k = state["rotary"](state["q"], state["k"], positions=state["positions"])
    if not c["train"]:
        return [q, k]
    return [q.detach(), k.detach(), *torch.autograd.grad([q, k], [state["q"], state["k"]], [state["dq"], state["dk"]])]


# --------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "ff":
        m, d, f = c["rows"], c["d"], c["ff"]
        values = m * d + 2 * f * d + m * f                       # x, both weights; h
        if c["train"]:
            values += m * f + m * d + 2 * f * d                  # dh; dx, both weight gradients
        return {"bytes": SIZE[c["dtype"]] * values, "flops": (12 if c["train"] else 4) * m * d * f}
    if c["op"] == "rope":
        rows = c["batch"] * c["len"]
        one = 2 * SIZE[c["dtype"]] * rows * (c["heads"] + c["kv"]) * c["head_dim"] + 8 * rows
        turned = rows * (c["heads"] + c["kv"]) * c["dim"]
        return {"bytes": one * (2 if c["train"] else 1), "flops": 3 * turned * (2 if c["train"] else 1)}
    sizes = _grad_sizes(c)
    once = sum(n * SIZE[k] for n, k in sizes)
    # gradients within the threshold stay as they are: one reading
    return {"bytes": once * (2 if _expected_norm(c) > c["max_norm"] else 1),
            "flops": 3 * sum(n for n, _ in sizes)}


# --------------------------------------------------------------------------- 64 bits
def _exact_ff(s, c):
    x, wg, wu = (s[k].detach().double() for k in ("x", "w_gate", "w_up"))
    gate, up = torch.einsum("md,fd->mf", x, wg), torch.einsum("md,fd->mf", x, wu)
    gate.requires_grad_()
    if c["act"] == "silu":
        a = gate * torch.sigmoid(gate)
    elif c["act"] == "gelu":
        a = gate * torch.special.ndtr(gate)
    else:
        a = gate * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate * gate * gate))
    if not c["train"]:
        return (a * up).detach()
    dh = s["dh"].double()
    (dgate,) = torch.autograd.grad(a, gate, dh * up)             # the derivative by autograd
    a = a.detach()
    dup = dh * a
    return [a * up, torch.einsum("mf,fd->md", dgate, wg) + torch.einsum("mf,fd->md", dup, wu),
            torch.einsum("mf,md->fd", dgate, x), torch.einsum("mf,md->fd", dup, x)]


def _exact_rope(s, c):
    freq, factor = _frequencies(c)
    spin = torch.polar(torch.full_like(freq, factor)[None, None, None],
                       (s["positions"].double()[:, None, :, None] * freq))
    n = freq.numel()

    def turned(x, spin):
        x = x.detach().double()
        head = x[..., :2 * n]
        pair = head.unflatten(-1, (n, 2)) if c["interleaved"] else head.unflatten(-1, (2, n)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * spin)
        z = z if c["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., 2 * n:]], dim=-1)

    out = [turned(s[k], spin) for k in ("q", "k")]
    if c["train"]:
        out += [turned(s[k], spin.conj()) for k in ("dq", "dk")]
    return out


def _exact_clip(s, c):
    # the flat buffers hold the gradients and, between them, zeros
    each = [f.double() for f in s["flats"]]
    norms = torch.stack([torch.linalg.vector_norm(f, ord=float(c["norm"])) for f in each])
    total = torch.linalg.vector_norm(norms, ord=float(c["norm"]))
    coef = torch.clamp(c["max_norm"] / (total + 1e-6), max=1.0)
    return [total] + [f * coef for f in each]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"ff": _exact_ff, "rope": _exact_rope, "clip": _exact_clip}[case["op"]](s, case)
