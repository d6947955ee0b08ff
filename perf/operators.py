"""Timed cases of the sequence operators in boltz_lumi_amd.ops.

Three operators that a sequence encoder / decoder beside the pair stack is
made of, each differentiable:

  rope      qk_norm_rope: RMS norm of every query and key head, then the
            rotation by position, both tensors in one pass
  relative  relative_bias: a learned bias by buckets of the distance
            k_pos - q_pos, [H, M, N], with the table's gradient
  attention cross_attention: queries of one sequence over the keys and values
            of another, with a key mask and an additive bias

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
THETA = 10000.0


# --------------------------------------------------------------------- cases


def listed():
    return [
        # one new token of a decoder: its query and key heads, where latency is all
        {"name": "rope_token", "kind": "rope", "type": "bf16", "batch": 1, "m": 1, "n": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "train": False, "start": 70001},
        # two long prompts, queries and keys of every head: a copy's worth of bytes
        {"name": "rope_prompt", "kind": "rope", "type": "bf16", "batch": 2, "m": 4096, "n": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "train": False, "start": 0},
        # training in fp32 with the token transformer's 16 x 48 heads, part of each head rotated, odd lengths
        {"name": "rope_train_fp32", "kind": "rope", "type": "fp32", "batch": 5, "m": 1134, "n": 577, "heads": 16,
         "kv_heads": 16, "dim": 48, "rotary": 32, "interleaved": True, "train": True, "start": 0},
        # the bias row of one new token over everything before it
        {"name": "relative_token", "kind": "relative", "type": "bf16", "batch": 0, "m": 1, "n": 1531, "heads": 16,
         "buckets": 32, "exact": 16, "max_distance": 128, "bidirectional": False, "train": False, "gaps": False},
        # residue numbers with chain gaps, clipped at 32 either side: two structures, forward
        {"name": "relative_residues", "kind": "relative", "type": "fp32", "batch": 2, "m": 1134, "n": 1134, "heads": 16,
         "buckets": 66, "exact": 32, "max_distance": 32, "bidirectional": True, "train": False, "gaps": True},
        # a training step of an encoder's bias: forward and the table's gradient
        {"name": "relative_train", "kind": "relative", "type": "fp32", "batch": 0, "m": 2048, "n": 2048, "heads": 16,
         "buckets": 32, "exact": 8, "max_distance": 128, "bidirectional": True, "train": True, "gaps": False},
        # one query over a small target's 117 tokens, the sequence stack's 16 x 24 heads, fp32
        {"name": "attention_token_n117", "kind": "attention", "type": "fp32", "batch": 1, "m": 1, "n": 117, "heads": 16,
         "kv_heads": 16, "dim": 24, "bias": "none", "lengths": "full", "train": False},
        # a decoding step of 32 sequences, each over its own encoder's states, ragged
        {"name": "attention_token_batch", "kind": "attention", "type": "bf16", "batch": 32, "m": 1, "n": 4096,
         "heads": 32, "kv_heads": 8, "dim": 128, "bias": "none", "lengths": "ragged", "train": False},
        # inference with one pair bias for five samples, ragged states of an odd length
        {"name": "attention_bias", "kind": "attention", "type": "bf16", "batch": 5, "m": 1024, "n": 1531, "heads": 16,
         "kv_heads": 16, "dim": 64, "bias": "shared", "lengths": "ragged", "train": False},
        # the largest: a training step over long states, four query heads to a key head
        {"name": "attention_train", "kind": "attention", "type": "bf16", "batch": 2, "m": 2048, "n": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "bias": "none", "lengths": "full", "train": True},
        # a training step with a bias that the batch shares, whose gradient is the sum over it
        {"name": "attention_train_bias", "kind": "attention", "type": "bf16", "batch": 4, "m": 577, "n": 1024,
         "heads": 16, "kv_heads": 16, "dim": 64, "bias": "shared", "lengths": "ragged", "train": True},
        # a training step in fp32, a bias of its own per element
        {"name": "attention_train_fp32", "kind": "attention", "type": "fp32", "batch": 2, "m": 312, "n": 1134,
         "heads": 16, "kv_heads": 16, "dim": 48, "bias": "own", "lengths": "ragged", "train": True},
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
    kind = rng.choice(["rope", "relative", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "rope":
        dim = rng.choice([24, 32, 48, 64, 96, 128])
        kv = rng.choice([1, 2, 4, 8])
        return {"kind": kind, "type": dtype, "batch": rng.choice([1, 2, 5]), "m": _log_int(rng, 1, 4096),
                "n": _log_int(rng, 1, 4096), "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": dim,
                "rotary": rng.choice([dim, dim // 16 * 8]), "interleaved": rng.random() < 0.5,
                "train": rng.random() < 0.5, "start": rng.choice([0, 3, 130001])}
    if kind == "relative":
        bidirectional, clipped = rng.random() < 0.6, rng.random() < 0.3
        side = rng.choice([16, 33, 64] if bidirectional else [16, 32, 64])
        return {"kind": kind, "type": dtype, "batch": rng.choice([0, 0, 1, 2]), "m": _log_int(rng, 1, 2048),
                "n": _log_int(rng, 1, 2048), "heads": rng.choice([1, 4, 12, 16]),
                "buckets": 2 * side if bidirectional else side, "exact": side - 1 if clipped else side // 2,
                "max_distance": rng.choice([128, 200, 1000]), "bidirectional": bidirectional,
                "train": rng.random() < 0.5, "gaps": rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 8])
    few = rng.random() < 0.35  # decoding steps
    return {"kind": kind, "type": dtype, "batch": rng.choice([1, 2, 5, 32] if few else [1, 2, 4, 5]),
            "m": rng.choice([1, 1, 4]) if few else _log_int(rng, 17, 2048), "n": _log_int(rng, 1, 4096),
            "heads": kv * rng.choice([1, 2, 4]), "kv_heads": kv, "dim": rng.choice([24, 32, 48, 64, 96, 128]),
            "bias": rng.choice(["none", "shared", "own"]), "lengths": rng.choice(["full", "ragged", "ragged_empty"]),
            "train": not few and rng.random() < 0.5}


def _lengths(case):
    """Valid keys of each batch element: an even spread, one element of several
    without any where the case says so."""
    b, n = case["batch"], case["n"]
    if case["lengths"] == "full":
        return [n] * b
    out = [max(1, n - (i * n * 3) // (5 * b)) for i in range(b)]
    if case["lengths"] == "ragged_empty" and b > 1:
        out[-1] = 0
    return out


def work(case):
    size = SIZE[case["type"]]
    if case["kind"] == "rope":
        elements = case["batch"] * case["dim"] * (case["m"] * case["heads"] + case["n"] * case["kv_heads"])
        # forward: x in, y out; backward: x and dy in, dx out
        return {"bytes": elements * size * (5 if case["train"] else 2), "flops": elements * (25 if case["train"] else 8)}
    if case["kind"] == "relative":
        elements = max(case["batch"], 1) * case["heads"] * case["m"] * case["n"]
        return {"bytes": elements * size * (2 if case["train"] else 1), "flops": elements * (2 if case["train"] else 1)}
    b, m, n, h, hk, d = (case[key] for key in ("batch", "m", "n", "heads", "kv_heads", "dim"))
    seen = sum(_lengths(case))
    rows, keys, bias = b * m * h * d, seen * hk * d, {"none": 0, "shared": 1, "own": b}[case["bias"]] * h * m * n
    moved = 2 * rows + 2 * keys + bias
    if case["train"]:  # and q, o, do, k, v, bias in; dq, dk, dv, dbias out
        moved += 4 * rows + 2 * keys + 2 * b * n * hk * d + 2 * bias
    return {"bytes": moved * size, "flops": (14 if case["train"] else 4) * m * seen * h * d}


# -------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape, dtype, scale=1.0, shift=0.0):
    return torch.randn(*shape, generator=g, device=DEVICE).mul_(scale).add_(shift).to(dtype)


def prepare(case, seed):
    g, dtype, train = _generator(seed), TYPES[case["type"]], case["train"]
    state = {"case": case}

    def leaf(t):
        return t.requires_grad_(train)

    if case["kind"] == "rope":
        b, d = case["batch"], case["dim"]
        # projections of a normalised stream: heads of different scales
        state["q"] = leaf(_randn(g, b, case["m"], case["heads"], d, dtype=dtype, scale=1.7))
        state["k"] = leaf(_randn(g, b, case["n"], case["kv_heads"], d, dtype=dtype, scale=0.6))
        state["q_weight"] = leaf(_randn(g, d, dtype=dtype, scale=0.2, shift=1.0))
        state["k_weight"] = leaf(_randn(g, d, dtype=dtype, scale=0.2, shift=1.0))
        state["q_pos"] = torch.arange(case["m"], device=DEVICE) + case["start"]
        state["k_pos"] = torch.arange(case["n"], device=DEVICE) + case["start"]
        half = case["rotary"] // 2
        state["inv_freq"] = THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half)
        if train:
            state["dq_out"] = _randn(g, *state["q"].shape, dtype=dtype)
            state["dk_out"] = _randn(g, *state["k"].shape, dtype=dtype)
    elif case["kind"] == "relative":
        b, m, n = case["batch"], case["m"], case["n"]
        state["table"] = leaf(_randn(g, case["buckets"], case["heads"], dtype=dtype))

        def positions(length):
            lead = (b,) if b else ()
            if not case["gaps"]:
                return torch.arange(length, device=DEVICE).expand(*lead, length).contiguous()
            # residue numbers: steps of 1 with a chain break (a jump back or ahead) now and then
            steps = torch.ones(*lead, length, device=DEVICE, dtype=torch.int64)
            breaks = torch.rand(*lead, length, generator=g, device=DEVICE) < 0.01
            jumps = torch.randint(-300, 300, (*lead, length), generator=g, device=DEVICE)
            return torch.where(breaks, jumps, steps).cumsum(-1)

        state["k_pos"] = positions(n)
        # a single query row stands behind the last key; others start with the keys
        state["q_pos"] = positions(m) if m > 1 else state["k_pos"][..., -1:].contiguous() + 1
        if train:
            state["dbias"] = _randn(g, *((b,) if b else ()), case["heads"], m, n, dtype=dtype)
    else:
        b, m, n, h, hk, d = (case[key] for key in ("batch", "m", "n", "heads", "kv_heads", "dim"))
        state["q"] = leaf(_randn(g, b, m, h, d, dtype=dtype))
        state["k"] = leaf(_randn(g, b, n, hk, d, dtype=dtype))
        state["v"] = leaf(_randn(g, b, n, hk, d, dtype=dtype))
        state["bias"] = None
        if case["bias"] != "none":
            state["bias"] = leaf(_randn(g, 1 if case["bias"] == "shared" else b, h, m, n, dtype=dtype))
        state["mask"] = None
        if case["lengths"] != "full":
            state["mask"] = torch.arange(n, device=DEVICE) < torch.tensor(_lengths(case), device=DEVICE)[:, None]
        if train:
            state["dout"] = _randn(g, b, m, h, d, dtype=dtype)
    return state


# --------------------------------------------------------- the plain forms


def _rotate(x, cos, sin, interleaved):
    """Rotation of the first 2 * len(cos) channels of x [B, T, H, D]; cos and sin [T, 1, R]."""
    r = cos.shape[-1]
    body, rest = x[..., :2 * r], x[..., 2 * r:]
    a, b = (body[..., 0::2], body[..., 1::2]) if interleaved else (body[..., :r], body[..., r:])
    a, b = a * cos - b * sin, a * sin + b * cos
    body = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([body, rest], -1)


def _plain_rope(s):
    case, outs, grads, weight_grads = s["case"], [], [], []
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"].float()
        angle = s[name + "_pos"].double()[:, None] * s["inv_freq"].double()
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        outs.append(_rotate(x * r * w, cos, sin, case["interleaved"]).to(s[name].dtype))
        if case["train"]:
            dy = _rotate(s["d" + name + "_out"].float(), cos, -sin, case["interleaved"])
            xn = x * r
            weight_grads.append((dy * xn).sum((0, 1, 2)).to(w.dtype).to(s[name].dtype))
            dn = dy * w
            grads.append((r * (dn - xn * (dn * xn).mean(-1, keepdim=True))).to(s[name].dtype))
    return tuple(outs + grads + weight_grads)


def _thresholds(side, exact, max_distance):
    """Least distance of each bucket 1 .. side - 1 of one direction: bucket i < exact holds the distance i,
    bucket exact + k the distances n with (n / exact)^steps >= (max_distance / exact)^k, in whole numbers."""
    steps, out = side - exact, list(range(1, exact + 1))
    for k in range(1, steps):
        n = max(out[-1], int(exact * (max_distance / exact) ** (k / steps)) - 2)
        while n ** steps < exact ** (steps - k) * max_distance ** k:
            n += 1
        out.append(n)
    return out


def _plain_buckets(s):
    case = s["case"]
    d = s["k_pos"][..., None, :] - s["q_pos"][..., :, None]
    side = case["buckets"] // 2 if case["bidirectional"] else case["buckets"]
    edges = torch.tensor(_thresholds(side, case["exact"], case["max_distance"]), device=d.device)
    n = d.abs() if case["bidirectional"] else (-d).clamp(min=0)
    bucket = torch.bucketize(n, edges, right=True)
    return bucket + side * (d > 0) if case["bidirectional"] else bucket


def _plain_relative(s):
    case, table = s["case"], s["table"].float()
    bucket = _plain_buckets(s)
    bias = table[bucket].movedim(-1, -3).to(s["table"].dtype).contiguous()
    if not case["train"]:
        return bias
    hit = (bucket[..., None] == torch.arange(case["buckets"], device=bucket.device)).float()
    by_row = torch.matmul(s["dbias"].float().transpose(-3, -2).contiguous(), hit)  # [.., M, H, buckets]
    dtable = by_row.flatten(0, -3).sum(0, dtype=torch.float64).t()
    return bias, dtable.to(s["table"].dtype).contiguous()


def _plain_attention(s):
    case = s["case"]
    b, m, n, h, hk, d = (case[key] for key in ("batch", "m", "n", "heads", "kv_heads", "dim"))
    group, scale, dtype = h // hk, case["dim"] ** -0.5, s["q"].dtype
    q = s["q"].float().transpose(1, 2)                                                   # [B, H, M, D]
    k = s["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    v = s["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    logits = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if s["bias"] is not None:
        logits = logits + s["bias"].float()
    if s["mask"] is not None:
        keep = s["mask"][:, None, None, :]
        logits = logits.masked_fill(~keep, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    del logits
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, v)
    result = out.transpose(1, 2).to(dtype).contiguous()
    if not case["train"]:
        return result
    dout = s["dout"].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout).unflatten(1, (hk, group)).sum(2)
    ds = torch.matmul(dout, v.transpose(2, 3).contiguous())
    ds = p * (ds - (dout * out).sum(-1, keepdim=True))
    del p
    dq = torch.matmul(ds, k) * scale
    dk = (torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale).unflatten(1, (hk, group)).sum(2)
    grads = [t.transpose(1, 2).to(dtype).contiguous() for t in (dq, dk, dv)]
    if s["bias"] is not None:
        grads.append((ds.sum(0, keepdim=True) if case["bias"] == "shared" else ds).to(dtype))
    return (result, *grads)


# ------------------------------------------------------ the framework's calls


def _own_rope(ops, s):
    case = s["case"]
    q, k = ops.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["q_pos"], s["k_pos"], s["inv_freq"],
                            eps=EPS, interleaved=case["interleaved"])
    if not case["train"]:
        return q, k
    grads = torch.autograd.grad((q, k), (s["q"], s["k"], s["q_weight"], s["k_weight"]), (s["dq_out"], s["dk_out"]))
    return q.detach(), k.detach(), *grads


def _own_relative(ops, s):
    case = s["case"]
    bias = ops.relative_bias(s["table"], s["q_pos"], s["k_pos"], exact=case["exact"],
                             max_distance=case["max_distance"], bidirectional=case["bidirectional"])
    if not case["train"]:
        return bias
    return bias.detach(), *torch.autograd.grad(bias, s["table"], s["dbias"])


def _own_attention(ops, s):
    out = ops.cross_attention(s["q"], s["k"], s["v"], mask=s["mask"], bias=s["bias"])
    if not s["case"]["train"]:
        return out
    leaves = [s[name] for name in ("q", "k", "v", "bias") if s[name] is not None]
    return out.detach(), *torch.autograd.grad(out, leaves, s["dout"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        from boltz_lumi_amd import ops

        with torch.set_grad_enabled(state["case"]["train"]):
            return {"rope": _own_rope, "relative": _own_relative, "attention": _own_attention}[kind](ops, state)
    with torch.no_grad():
        return {"rope": _plain_rope, "relative": _plain_relative, "attention": _plain_attention}[kind](state)


# ---------------------------------------------------------------- in 64 bits


def _exact_rope(s):
    case, outs, grads, weight_grads = s["case"], [], [], []
    half = case["rotary"] // 2
    channel = torch.arange(half, device=DEVICE)
    first, second = (2 * channel, 2 * channel + 1) if case["interleaved"] else (channel, channel + half)
    for name in ("q", "k"):
        x, w = s[name].double(), s[name + "_weight"].double()
        angle = torch.outer(s[name + "_pos"].double(), s["inv_freq"].double())
        turn = torch.polar(torch.ones_like(angle), angle)[None, :, None]  # e^(i pos f)

        def rotated(t, factor):
            z = torch.complex(t[..., first], t[..., second]) * factor
            t = t.clone()
            t[..., first], t[..., second] = z.real, z.imag
            return t

        norm = (x.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
        outs.append(rotated(x / norm * w, turn))
        if case["train"]:
            g = rotated(s["d" + name + "_out"].double(), turn.conj())
            weight_grads.append((g * x / norm).flatten(0, 2).sum(0))
            gw = g * w
            grads.append(gw / norm - x * (gw * x).sum(-1, keepdim=True) / (case["dim"] * norm ** 3))
    return tuple(outs + grads + weight_grads)


def _exact_relative(s):
    case = s["case"]
    side = case["buckets"] // 2 if case["bidirectional"] else case["buckets"]
    e, top = case["exact"], case["max_distance"]

    def bucket(n):  # of a distance in one direction, from its definition in whole numbers
        if n < e:
            return n
        return e + max(k for k in range(side - e) if n ** (side - e) >= e ** (side - e - k) * top ** k)

    far = max(e, top) + 1  # every distance from here on is in the last bucket
    of = torch.tensor([bucket(n) for n in range(far + 1)], device=DEVICE)
    d = s["k_pos"].unsqueeze(-2) - s["q_pos"].unsqueeze(-1)
    if case["bidirectional"]:
        index = of[d.abs().clamp(max=far)] + torch.where(d > 0, side, 0)
    else:
        index = of[d.neg().clamp(0, far)]
    table = s["table"].double()
    bias = torch.stack([table[:, i][index] for i in range(case["heads"])], -3)
    if not case["train"]:
        return bias
    dtable = torch.zeros_like(table)
    for i in range(case["heads"]):
        dtable[:, i].index_add_(0, index.flatten(), s["dbias"].select(-3, i).double().flatten())
    return bias, dtable


def _exact_attention(s):
    case = s["case"]
    b, m, n, h, hk, d = (case[key] for key in ("batch", "m", "n", "heads", "kv_heads", "dim"))
    lengths = _lengths(case)

    def zeros(name):
        return torch.zeros(s[name].shape, device=DEVICE, dtype=torch.float64)

    out, dq, dk, dv = zeros("q"), zeros("q"), zeros("k"), zeros("v")
    dbias = None if s["bias"] is None else zeros("bias")
    for i in range(b):
        keys = lengths[i]
        if not keys:
            continue
        for j in range(h):
            q, k, v = s["q"][i, :, j].double(), *(s[t][i, :keys, j * hk // h].double() for t in ("k", "v"))
            logits = q @ k.T / math.sqrt(d)
            if dbias is not None:
                at = (i if case["bias"] == "own" else 0, j)
                logits += s["bias"][at][:, :keys].double()
            weights = torch.softmax(logits, -1)
            out[i, :, j] = weights @ v
            if not case["train"]:
                continue
            g = s["dout"][i, :, j].double()
            dv[i, :keys, j * hk // h] += weights.T @ g
            back = g @ v.T
            back = weights * (back - (weights * back).sum(-1, keepdim=True))
            dq[i, :, j] = back @ k / math.sqrt(d)
            dk[i, :keys, j * hk // h] += back.T @ q / math.sqrt(d)
            if dbias is not None:
                dbias[at][:, :keys] += back
    if not case["train"]:
        return out
    return (out, dq, dk, dv) if dbias is None else (out, dq, dk, dv, dbias)


def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        return {"rope": _exact_rope, "relative": _exact_relative, "attention": _exact_attention}[case["kind"]](state)
