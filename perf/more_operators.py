"""Timed cases of the sequence mixing operators in boltz_lumi_amd.ops.

Three operators that a block of a sequence stack is made of whose cost is linear
in the tokens, each differentiable, each with its form for single tokens:

  norm   residual_norm: RMS norm of a block's result, its gate and residual
         scale, the residual add and the next block's RMS norm, one pass
  conv   causal_conv: short causal convolution of every channel with SiLU,
         carrying the last inputs from call to call
  scan   selective_scan: a diagonal state space whose step, input and output
         maps depend on the token, carrying its state from call to call

``prepare`` makes what a program holds before the call, ``run`` is one pass
(the plain form in 32 bits, or the framework's kernels where ``own`` is set),
``exact`` the same outputs in 64 bits, ``work`` the bytes and operations that a
pass cannot do without.  A case with "train" returns the gradients too.
"""

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}
EPS = 1e-6


# --------------------------------------------------------------------- cases


def listed():
    return [
        # a decoding step of 32 sequences: the residual frame between two blocks, where latency is all
        {"name": "norm_token", "kind": "norm", "stream": "bf16", "type": "bf16", "batch": 32, "tokens": 1, "dim": 768,
         "gate": "token", "train": False},
        # two long prompts on an fp32 residual stream with bf16 blocks: a copy's worth of bytes
        {"name": "norm_prompt", "kind": "norm", "stream": "fp32", "type": "bf16", "batch": 2, "tokens": 8192, "dim": 2048,
         "gate": "token", "train": False},
        # training at the token transformer's width, five samples, one gate per sample (its conditioning), odd length
        {"name": "norm_train_fp32", "kind": "norm", "stream": "fp32", "type": "fp32", "batch": 5, "tokens": 1134,
         "dim": 768, "gate": "sample", "train": True},
        # training of a wide stack on the fp32 stream
        {"name": "norm_train", "kind": "norm", "stream": "fp32", "type": "bf16", "batch": 4, "tokens": 2048, "dim": 2048,
         "gate": "token", "train": True},
        # a decoding step: 32 sequences' last inputs move on by one token
        {"name": "conv_token", "kind": "conv", "type": "bf16", "batch": 32, "tokens": 1, "channels": 1536, "width": 4,
         "lengths": "full", "state": True, "train": False},
        # one long fp32 chain read in two parts, the second with the first one's last inputs
        {"name": "conv_long_fp32", "kind": "conv", "type": "fp32", "batch": 1, "tokens": 16001, "channels": 768, "width": 3,
         "lengths": "full", "state": True, "train": False},
        # a training step over ragged sequences
        {"name": "conv_train", "kind": "conv", "type": "bf16", "batch": 4, "tokens": 2048, "channels": 1536, "width": 4,
         "lengths": "ragged", "state": False, "train": True},
        # a decoding step: 32 sequences' states move on by one token
        {"name": "scan_token", "kind": "scan", "type": "bf16", "batch": 32, "tokens": 1, "channels": 1536, "states": 16,
         "groups": 1, "gate": True, "lengths": "full", "state": True, "train": False},
        # two prompts of different lengths, whose last states start the decoding
        {"name": "scan_prompt", "kind": "scan", "type": "bf16", "batch": 2, "tokens": 4096, "channels": 1536, "states": 16,
         "groups": 1, "gate": True, "lengths": "ragged", "state": True, "train": False},
        # one long chain of few channels in fp32: only its length can fill the card
        {"name": "scan_long_fp32", "kind": "scan", "type": "fp32", "batch": 1, "tokens": 16001, "channels": 384,
         "states": 8, "groups": 1, "gate": False, "lengths": "full", "state": False, "train": False},
        # the largest: a training step over ragged sequences
        {"name": "scan_train", "kind": "scan", "type": "bf16", "batch": 4, "tokens": 2048, "channels": 1536, "states": 16,
         "groups": 1, "gate": True, "lengths": "ragged", "state": False, "train": True},
        # training in fp32 of a part of longer sequences: four groups of channels, many states, carried over
        {"name": "scan_train_groups_fp32", "kind": "scan", "type": "fp32", "batch": 2, "tokens": 577, "channels": 384,
         "states": 64, "groups": 4, "gate": True, "lengths": "full", "state": True, "train": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _fits(case):
    """No more than the largest listed case of the kind costs."""
    most = {"bytes": 0, "flops": 0}
    for other in listed():
        if other["kind"] == case["kind"]:
            w = work(other)
            most = {key: max(most[key], w[key]) for key in most}
    w = work(case)
    return all(w[key] <= most[key] for key in most)


def draw(rng):
    while True:
        case = _draw(rng)
        if _fits(case):
            return case


def _draw(rng):
    kind = rng.choice(["norm", "conv", "scan", "scan"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    token, train = rng.random() < 0.2, rng.random() < 0.5  # a decoding step takes no gradient
    batch = rng.choice([1, 2, 8, 32]) if token else rng.choice([1, 2, 4, 5])
    if kind == "norm":
        return {"kind": kind, "stream": "fp32" if dtype == "fp32" else rng.choice(["bf16", "fp32"]), "type": dtype,
                "batch": batch, "tokens": 1 if token else _log_int(rng, 1, 8192), "dim": 8 * _log_int(rng, 1, 1024),
                "gate": rng.choice(["none", "token", "sample"]), "train": train and not token}
    case = {"kind": kind, "type": dtype, "batch": batch, "lengths": rng.choice(["full", "ragged", "ragged_empty"]),
            "state": token or rng.random() < 0.5, "train": train and not token}
    if token:
        case["lengths"] = "full"
    if kind == "conv":
        return {**case, "tokens": 1 if token else _log_int(rng, 1, 16384), "channels": 8 * _log_int(rng, 1, 256),
                "width": rng.choice([2, 3, 4])}
    groups = rng.choice([1, 1, 2, 4])
    return {**case, "tokens": 1 if token else _log_int(rng, 1, 4096 if case["train"] else 16384),
            "channels": 8 * groups * _log_int(rng, 1, 256 // groups), "states": rng.choice([8, 16, 16, 32, 64]),
            "groups": groups, "gate": rng.random() < 0.7}


def _lengths(case):
    """Tokens of each batch element: an even spread, one element of several
    without any where the case says so."""
    b, t = case["batch"], case["tokens"]
    if case["lengths"] == "full":
        return [t] * b
    out = [max(1, t - (i * t * 3) // (5 * b)) for i in range(b)]
    if case["lengths"] == "ragged_empty" and b > 1:
        out[-1] = 0
    return out


def work(case):
    size, train = SIZE[case["type"]], case["train"]
    if case["kind"] == "norm":
        rows, d, stream = case["batch"] * case["tokens"], case["dim"], SIZE[case["stream"]]
        gates = {"none": 0, "token": rows, "sample": case["batch"]}[case["gate"]] * d * size
        moved = rows * d * 2 * (stream + size) + gates  # x, y in; r, h out
        if train:  # x, y, dr, dh in; dx, dy out
            moved += rows * d * 3 * (stream + size) + 2 * gates
        return {"bytes": moved, "flops": rows * d * (45 if train else 15)}
    seen = sum(_lengths(case))
    if case["kind"] == "conv":
        c, w = case["channels"], case["width"]
        state = 2 * case["batch"] * (w - 1) * c * size if case["state"] else 0
        return {"bytes": seen * c * size * (5 if train else 2) + state * (2 if train else 1),
                "flops": seen * c * ((6 * w + 15) if train else (2 * w + 5))}
    c, n, g = case["channels"], case["states"], case["groups"]
    rows, maps = seen * c * size, 2 * seen * g * n * size
    state = 2 * case["batch"] * c * n * 4 if case["state"] else 0
    moved = rows * (4 if case["gate"] else 3) + maps + state  # u, dt, (z), B, C in; y out
    if train:  # u, dt, (z), dy, B, C in; du, ddt, (dz), dB, dC out
        moved += rows * (7 if case["gate"] else 5) + 2 * maps + state
    # a state of a channel and token: the decay's product and exp, the input, two multiply-adds (7); backward the same
    # state again (5), the gradient's recurrence and six sums (17)
    return {"bytes": moved, "flops": seen * c * n * (29 if train else 7)}


# -------------------------------------------------------------------- inputs


def _randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=g, device=DEVICE).mul_(scale).add_(shift).to(dtype)


def prepare(case, seed):
    g, dtype, train = torch.Generator(device=DEVICE).manual_seed(seed), TYPES[case["type"]], case["train"]
    state, b, t = {"case": case}, case["batch"], case["tokens"]

    def leaf(value):
        return value.requires_grad_(train)

    if case["kind"] == "norm":
        d, stream = case["dim"], TYPES[case["stream"]]
        # a stream that has grown over the blocks before, a block's result of another size
        state["x"] = leaf(_randn(g, b, t, d, dtype=stream, scale=3.0))
        state["y"] = leaf(_randn(g, b, t, d, dtype=dtype, scale=0.7))
        state["gate"] = None
        if case["gate"] != "none":
            state["gate"] = leaf(_randn(g, b, t if case["gate"] == "token" else 1, d, dtype=dtype))
        state["y_weight"] = leaf(_randn(g, d, scale=0.2, shift=1.0))
        state["scale"] = leaf(_randn(g, d, scale=0.1, shift=0.3))
        state["weight"] = leaf(_randn(g, d, scale=0.2, shift=1.0))
        if train:
            state["dr"] = _randn(g, b, t, d, dtype=stream)
            state["dh"] = _randn(g, b, t, d, dtype=dtype)
        return state
    c = case["channels"]
    state["lengths"] = None
    if case["lengths"] != "full":
        state["lengths"] = torch.tensor(_lengths(case), device=DEVICE)
    state["first"] = state["next"] = state["dnext"] = None
    if case["kind"] == "conv":
        w = case["width"]
        state["x"] = leaf(_randn(g, b, t, c, dtype=dtype))
        state["weight"] = leaf(_randn(g, c, w, scale=w ** -0.5))
        state["bias"] = leaf(_randn(g, c, scale=0.1))
        if case["state"]:
            state["first"] = leaf(_randn(g, b, w - 1, c, dtype=dtype))
    else:
        n, groups = case["states"], case["groups"]
        state["u"] = leaf(_randn(g, b, t, c, dtype=dtype))
        state["dt"] = leaf(_randn(g, b, t, c, dtype=dtype, scale=0.5))
        # decays from one over the number of a channel's states, steps from 0.001 to 0.1
        state["A"] = leaf(-(torch.arange(1, n + 1, device=DEVICE) * torch.exp(_randn(g, c, n, scale=0.1))))
        step = torch.exp(torch.rand(c, generator=g, device=DEVICE) * math.log(100.0) + math.log(0.001))
        state["dt_bias"] = leaf(step + torch.log(-torch.expm1(-step)))
        state["B"] = leaf(_randn(g, b, t, groups, n, dtype=dtype))
        state["C"] = leaf(_randn(g, b, t, groups, n, dtype=dtype))
        state["D"] = leaf(_randn(g, c, scale=0.1, shift=1.0))
        state["z"] = leaf(_randn(g, b, t, c, dtype=dtype)) if case["gate"] else None
        if case["state"]:
            state["first"] = leaf(_randn(g, b, c, n, scale=0.3))
    if case["state"] and train:
        state["dnext"] = _randn(g, *state["first"].shape, dtype=state["first"].dtype)
    elif case["state"]:
        state["next"] = torch.empty_like(state["first"])  # where a decoder keeps it
    if train:
        state["dy"] = _randn(g, b, t, c, dtype=dtype)
    return state


# --------------------------------------------------------- the plain forms


def _plain_norm(s):
    case = s["case"]
    x, y, yw, scale, w = (s[name].float() for name in ("x", "y", "y_weight", "scale", "weight"))
    gate = torch.sigmoid(s["gate"].float()) if s["gate"] is not None else torch.ones((), device=x.device)
    rho_y = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    n = y * rho_y
    m = n * yw
    r = x + scale * gate * m
    rho_r = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    r_hat = r * rho_r
    result = r.to(s["x"].dtype), (r_hat * w).to(s["y"].dtype)
    if not case["train"]:
        return result

    def over_rows(v):
        return v.sum((0, 1), dtype=torch.float64).float()

    dh = s["dh"].float()
    e = dh * w
    dr = s["dr"].float() + rho_r * (e - r_hat * (e * r_hat).mean(-1, keepdim=True))
    dw = over_rows(dh * r_hat)
    back = dr * gate
    dscale = over_rows(back * m)
    dyw = over_rows(back * scale * n)
    f = back * scale * yw
    dy = rho_y * (f - n * (f * n).mean(-1, keepdim=True))
    grads = [dr.to(s["x"].dtype), dy.to(s["y"].dtype)]
    if s["gate"] is not None:
        dgate = back * scale * m * (1 - gate)
        if case["gate"] == "sample":
            dgate = dgate.sum(1, keepdim=True, dtype=torch.float64)
        grads.append(dgate.to(s["gate"].dtype))
    return (*result, *grads, dyw, dscale, dw)


def _keep(s):
    """1 for the tokens of each sequence, 0 behind its end: [B, T, 1]."""
    case = s["case"]
    if s["lengths"] is None:
        return torch.ones(1, 1, 1, device=DEVICE)
    return (torch.arange(case["tokens"], device=DEVICE) < s["lengths"][:, None]).float()[..., None]


def _plain_conv(s):
    case, dtype = s["case"], s["x"].dtype
    b, t, c, width = case["batch"], case["tokens"], case["channels"], case["width"]
    x, w, keep = s["x"].float(), s["weight"].float(), _keep(s)
    first = s["first"].float() if s["first"] is not None else x.new_zeros(b, width - 1, c)
    rows = torch.cat([first, x], 1)
    p = s["bias"].float() + sum(w[:, j] * rows[:, j:j + t] for j in range(width))
    gate = torch.sigmoid(p)
    result = [(p * gate * keep).to(dtype)]
    if case["state"]:
        end = s["lengths"] if s["lengths"] is not None else torch.full((b,), t, device=x.device)
        at = (end[:, None] + torch.arange(width - 1, device=x.device))[..., None].expand(-1, -1, c)
        result.append(rows.gather(1, at).to(dtype))
    if not case["train"]:
        return tuple(result)
    dp = s["dy"].float() * (gate + p * gate * (1 - gate)) * keep
    drows = torch.zeros_like(rows)
    if case["state"]:
        drows.scatter_(1, at, s["dnext"].float())
    for j in range(width):
        drows[:, j:j + t] += dp * w[:, j]
    dw = torch.stack([(dp * rows[:, j:j + t]).sum((0, 1), dtype=torch.float64) for j in range(width)], 1).float()
    grads = [drows[:, width - 1:].to(dtype), dw, dp.sum((0, 1), dtype=torch.float64).float()]
    if case["state"]:
        grads.append(drows[:, :width - 1].to(dtype))
    return (*result, *grads)


def _scan(a, v):
    """h[t] = a[t] h[t - 1] + v[t] along the first axis, by doubling: log2(T) elementwise steps over all tokens."""
    k = 1
    while k < v.shape[0]:
        v = torch.cat([v[:k], v[k:] + a[k:] * v[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return v


def _plain_scan(s):
    case, dtype = s["case"], s["u"].dtype
    b, t, c, n, groups = (case[key] for key in ("batch", "tokens", "channels", "states", "groups"))
    u, dt, keep = (v.transpose(0, 1) for v in (s["u"].float(), s["dt"].float() + s["dt_bias"], _keep(s)))  # [T, B, C]
    A = s["A"]
    Bm, Cm = (s[name].float().transpose(0, 1).unsqueeze(3).expand(-1, -1, -1, c // groups, -1).flatten(2, 3)
              for name in ("B", "C"))  # [T, B, C, N]
    first = s["first"] if s["first"] is not None else u.new_zeros(b, c, n)
    delta = (dt.clamp(min=0) + torch.log1p(torch.exp(-dt.abs()))) * keep
    a = torch.exp(delta[..., None] * A)
    v = (delta * u)[..., None] * Bm
    v[0] += a[0] * first
    h = _scan(a, v)
    del v
    y = (h * Cm).sum(-1) + s["D"] * u
    z = s["z"].float().transpose(0, 1) if case["gate"] else None
    sig = torch.sigmoid(z) if case["gate"] else None
    out = (y * z * sig if case["gate"] else y) * keep
    result = [out.transpose(0, 1).to(dtype).contiguous()]
    if case["state"]:
        result.append(h[-1].clone())
    if not case["train"]:
        return tuple(result)

    def rows(value):
        return value.transpose(0, 1).to(dtype).contiguous()

    def over_tokens(value):
        return value.sum((0, 1), dtype=torch.float64).float()

    def over_channels(value):  # [T, B, C, N] to [B, T, G, N]
        return rows(value.unflatten(2, (groups, c // groups)).sum(3))

    dout = s["dy"].float().transpose(0, 1) * keep
    dy = dout * z * sig if case["gate"] else dout
    back = dy[..., None] * Cm
    if case["state"]:
        back[-1] += s["dnext"]
    after = torch.cat([a[1:], torch.zeros_like(a[:1])])
    G = _scan(after.flip(0), back.flip(0)).flip(0)
    del after, back
    dC = over_channels(dy[..., None] * h)
    dB = over_channels(G * (delta * u)[..., None])
    q = G * a * torch.cat([first[None], h[:-1]])
    GB = (G * Bm).sum(-1)
    du = delta * GB + s["D"] * dy
    dA = over_tokens(q * delta[..., None])
    ddt = ((q * A).sum(-1) + u * GB) * torch.sigmoid(dt) * keep
    grads = [rows(du), rows(ddt), dA, dB, dC, over_tokens(dy * u), over_tokens(ddt)]
    if case["gate"]:
        grads.append(rows(dout * y * (sig + z * sig * (1 - sig))))
    if case["state"]:
        grads.append(a[0] * G[0])
    return (*result, *grads)


# ------------------------------------------------------ the framework's calls


def _own_norm(ops, s):
    case = s["case"]
    r, h = ops.residual_norm(s["x"], s["y"], s["gate"], s["y_weight"], s["scale"], s["weight"], eps=EPS)
    if not case["train"]:
        return r, h
    leaves = [s[name] for name in ("x", "y", "gate", "y_weight", "scale", "weight") if s[name] is not None]
    return r.detach(), h.detach(), *torch.autograd.grad((r, h), leaves, (s["dr"], s["dh"]))


def _with_state(s, result, names):
    """The results of a call that may carry a state, and the gradients where the case trains."""
    case = s["case"]
    results = result if case["state"] else (result,)
    if not case["train"]:
        return tuple(results)
    leaves = [s[name] for name in names if s[name] is not None]
    given = (s["dy"], s["dnext"]) if case["state"] else (s["dy"],)
    return *(r.detach() for r in results), *torch.autograd.grad(results, leaves, given)


def _own_conv(ops, s):
    result = ops.causal_conv(s["x"], s["weight"], s["bias"], state=s["first"], lengths=s["lengths"],
                             return_state=s["case"]["state"], state_out=s["next"])
    return _with_state(s, result, ("x", "weight", "bias", "first"))


def _own_scan(ops, s):
    result = ops.selective_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["z"], s["dt_bias"], state=s["first"],
                                lengths=s["lengths"], return_state=s["case"]["state"], state_out=s["next"])
    return _with_state(s, result, ("u", "dt", "A", "B", "C", "D", "dt_bias", "z", "first"))


def run(state):
    kind = state["case"]["kind"]
    if own:
        from boltz_lumi_amd import ops

        with torch.set_grad_enabled(state["case"]["train"]):
            return {"norm": _own_norm, "conv": _own_conv, "scan": _own_scan}[kind](ops, state)
    with torch.no_grad():
        return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan}[kind](state)


# ---------------------------------------------------------------- in 64 bits
#
# The forward pass from its definition, element after element and token after
# token, and the gradients by differentiating that.


def _exact_norm(s, v):
    norm_y = (v["y"].square().sum(-1, keepdim=True) / s["case"]["dim"] + EPS).sqrt()
    block = v["y"] / norm_y * v["y_weight"] * v["scale"]
    if v["gate"] is not None:
        block = block / (1 + torch.exp(-v["gate"]))
    r = v["x"] + block
    return r, r / (r.square().sum(-1, keepdim=True) / s["case"]["dim"] + EPS).sqrt() * v["weight"]


def _exact_conv(s, v):
    case, outs, states = s["case"], [], []
    width, c = case["width"], case["channels"]
    for i, end in enumerate(_lengths(case)):
        seen = v["x"].new_zeros(width - 1, c) if v["first"] is None else v["first"][i]
        seen = torch.cat([seen, v["x"][i, :end]])
        taps = seen.unfold(0, width, 1) if end else seen.new_zeros(0, c, width)  # [end, C, W]
        p = (taps * v["weight"]).sum(-1) + v["bias"]
        outs.append(torch.cat([p / (1 + torch.exp(-p)), p.new_zeros(case["tokens"] - end, c)]))
        states.append(seen[end:])
    out = torch.stack(outs)
    return (out, torch.stack(states)) if case["state"] else (out,)


def _exact_scan(s, v):
    case, outs, states = s["case"], [], []
    c, n, repeat = case["channels"], case["states"], case["channels"] // case["groups"]
    for i, end in enumerate(_lengths(case)):
        h = v["A"].new_zeros(c, n) if v["first"] is None else v["first"][i]
        ys = []
        steps = torch.log1p(torch.exp(v["dt"][i] + v["dt_bias"])).unbind(0)
        us, maps_in, maps_out = v["u"][i].unbind(0), v["B"][i].unbind(0), v["C"][i].unbind(0)
        for j in range(end):
            into = steps[j] * us[j]
            h = torch.exp(steps[j][:, None] * v["A"]) * h + into[:, None] * maps_in[j].repeat_interleave(repeat, 0)
            ys.append((h * maps_out[j].repeat_interleave(repeat, 0)).sum(-1))
        if end:
            y = torch.stack(ys) + v["D"] * v["u"][i, :end]
            if case["gate"]:
                y = y * v["z"][i, :end] / (1 + torch.exp(-v["z"][i, :end]))
            ys = [y]
        outs.append(torch.cat([*ys, v["u"].new_zeros(case["tokens"] - end, c)]))
        states.append(h)
    out = torch.stack(outs)
    return (out, torch.stack(states)) if case["state"] else (out,)


def exact(case, seed):
    if case["kind"] == "scan" and sum(_lengths(case)) > (12000 if case["train"] else 40000):
        return None  # too many steps one by one
    s, train = prepare(case, seed), case["train"]
    form, names, given = {
        "norm": (_exact_norm, ("x", "y", "gate", "y_weight", "scale", "weight"), ("dr", "dh")),
        "conv": (_exact_conv, ("x", "weight", "bias", "first"), ("dy", "dnext")),
        "scan": (_exact_scan, ("u", "dt", "A", "B", "C", "D", "dt_bias", "z", "first"), ("dy", "dnext")),
    }[case["kind"]]
    v = {name: None if s[name] is None else s[name].detach().double().requires_grad_(train) for name in names}
    with torch.set_grad_enabled(train):
        results = form(s, v)
        if not train:
            return tuple(results)
        leaves = [v[name] for name in names if v[name] is not None]
        back = [s[name].double() for name in given if s[name] is not None]
        grads = torch.autograd.grad(results, leaves, back, allow_unused=True)
    return *(r.detach() for r in results), *(torch.zeros_like(x) if d is None else d for d, x in zip(grads, leaves))
