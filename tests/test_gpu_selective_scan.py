"""ops.selective_scan and its gradients against the oracle in fp64.

Tolerances: half a step of the result's type, and roundings of 2^-24 relative to the magnitudes that a value is made of.
A term of a result goes through at most T tokens; each multiplies it by a decay exp2(d A log2(e)), whose exponent (below 8
here) is rounded twice and which the hardware gives to one step (2 roundings), and adds it to a sum: under 8 roundings
where the exponent is at most 2 (where it is larger, what is left of the term is smaller by more).  Everything else (the
step, the maps, sums over 64 states, the gate and its slope) is under 96; a sum over rows adds at most one a row."""

import pytest
import torch

from boltz_lumi_amd import ops
from oracle import mixing
from mixing_cases import BF16, FP32, assert_close, fp64, leaf, randn

pytestmark = pytest.mark.gpu

NAMES = ["out", "state", "du", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dstate"]


def make(b, t, c, n, groups, dtype, absent="", softplus=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    u, z = randn(g, b, t, c, dtype=dtype), randn(g, b, t, c, dtype=dtype)
    dt = randn(g, b, t, c, dtype=dtype) if softplus else randn(g, b, t, c, scale=0.05, dtype=FP32).abs().to(dtype)
    A = -(randn(g, c, n).abs() + 0.1)
    B, C = (randn(g, b, t, groups, n, dtype=dtype) for _ in range(2))
    D, bias = randn(g, c), randn(g, c, scale=0.5, shift=-2.0) if softplus else randn(g, c, scale=0.01).abs()
    inputs = [u, dt, A, B, C, D, z, bias, randn(g, b, c, n)]
    for i, letter in ((5, "D"), (6, "z"), (7, "b"), (8, "s")):
        if letter in absent:
            inputs[i] = None
    return inputs, [randn(g, b, t, c, dtype=dtype), randn(g, b, c, n)]


def call(v, lengths=None, softplus=True, **more):
    return ops.selective_scan(*v[:8], state=v[8], lengths=lengths, softplus=softplus, **more)


def check(inputs, back, gpu, lengths=None, softplus=True, view=lambda t: t, index=torch.int64):
    leaves = [leaf(t, gpu) for t in inputs]
    b, t, c = inputs[0].shape
    on_gpu = None if lengths is None else torch.tensor(lengths, device=gpu, dtype=index)
    seen = [None if x is None else view(x) if x.dim() > 2 and i != 8 else x for i, x in enumerate(leaves)]
    made = call(seen, on_gpu, softplus, return_state=True)
    grads = iter(torch.autograd.grad(made, [x for x in leaves if x is not None], [x.to(gpu) for x in back]))
    got = [*made, *(None if x is None else next(grads) for x in leaves)]
    ends = [t] * b if lengths is None else [min(max(k, 0), t) for k in lengths]
    with torch.no_grad():
        results, sizes = mixing.selective_scan(*map(fp64, inputs), ends, softplus, *map(fp64, back))
    for name, a, w, size in zip(NAMES, got, results, sizes):
        rows = b * t if name in ("dA", "dD", "ddt_bias") else c if name in ("dB", "dC") else 0
        assert_close(name, a, w, size, 96 + 8 * max(ends, default=0) + rows)
    return got


@pytest.mark.parametrize("t", [1, 2, 3, 4, 5, 31, 32, 33, 64, 65, 100])
@pytest.mark.parametrize("n", [8, 16, 32, 64])
def test_tokens_and_states(gpu, t, n):
    check(*make(2, t, 16, n, 1, BF16, seed=t), gpu)


@pytest.mark.parametrize("c,groups", [(8, 1), (24, 3), (40, 1), (64, 1), (72, 1), (200, 5), (264, 1)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_channels_and_groups(gpu, c, groups, dtype):
    check(*make(2, 37, c, 16, groups, dtype, seed=c), gpu)


@pytest.mark.parametrize("c,n", [(1000, 8), (408, 16), (392, 32), (200, 64)])
def test_spans(gpu, c, n):
    """More channels than a gradient block's: dB and dC are added over several."""
    check(*make(1, 35, c, n, 1, FP32, seed=c), gpu)
    check(*make(2, 33, 2 * c, n, 2, BF16, seed=c), gpu)


@pytest.mark.parametrize("absent", ["D", "z", "b", "s", "Dz", "Dzbs"])
@pytest.mark.parametrize("softplus", [True, False])
def test_absent_parts(gpu, absent, softplus):
    check(*make(2, 41, 24, 16, 1, FP32, absent, softplus), gpu, softplus=softplus)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [8, 32])
def test_ragged(gpu, index, n):
    """Lengths of nothing, one, around the tiles, to the end and past both ends; what stands behind them is NaN and unseen."""
    lengths = [0, 1, 31, 32, 33, 64, 70, 99, -5]
    inputs, back = make(9, 70, 16, n, 2, BF16)
    for i, k in enumerate(lengths):
        for t in (*(inputs[j] for j in (0, 1, 3, 4, 6)), back[0]):
            t[i, max(k, 0):] = float("nan")
    got = check(inputs, back, gpu, lengths, index=index)
    for i, k in enumerate(lengths):
        assert all(not got[j][i, max(k, 0):].any() for j in (0, 2, 3, 5, 6, 8))
        if k <= 0:
            assert torch.equal(got[1][i].cpu(), inputs[8][i]) and torch.equal(got[10][i].cpu(), back[1][i])


def test_strides(gpu):
    inputs, back = make(3, 9, 32, 16, 2, BF16)

    def slices(t):
        width = t.shape[-1]
        wide = torch.full((*t.shape[:-1], 3 * width), float("nan"), device=t.device, dtype=t.dtype)
        wide[..., width:2 * width] = t
        return wide[..., width:2 * width]

    for view in (slices, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: t.transpose(1, -1).contiguous().transpose(1, -1),
                 lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)):
        check(inputs, back, gpu, view=view)
        leaves = [None if x is None else view(x.to(gpu)) if x.dim() > 2 and i != 8 else x.to(gpu)
                  for i, x in enumerate(inputs)]
        one = [x[:, :1] if i in (0, 1, 3, 4, 6) else x for i, x in enumerate(leaves)]
        assert torch.equal(call(one), call([x.contiguous() for x in one]))


@pytest.mark.parametrize("shape", ["broadcast", "packed"])
def test_shared_operands(gpu, shape):
    """Maps that the batch shares (stride 0), whose gradients torch adds; everything in one projection's columns."""
    inputs, back = make(2, 40, 16, 8, 1, FP32)
    if shape == "broadcast":
        for i in (3, 4):
            inputs[i][1] = inputs[i][0]
        leaves = [leaf(t[:1] if i in (3, 4) else t, gpu) for i, t in enumerate(inputs)]
        seen = [t.expand(2, -1, -1, -1) if i in (3, 4) else t for i, t in enumerate(leaves)]
        made = call(seen, return_state=True)
        got = torch.autograd.grad(made, leaves[3:5], [t.to(gpu) for t in back])
        with torch.no_grad():
            results, sizes = mixing.selective_scan(*map(fp64, inputs), [40, 40], True, *map(fp64, back))
        for a, w, size in zip(got, results[5:7], sizes[5:7]):
            assert_close("maps", a, w.sum(0, keepdim=True), size.sum(0, keepdim=True), 96 + 8 * 40 + 16 + 2)
    else:
        u, dt, _, B, C, _, z, _, _ = inputs
        packed = leaf(torch.cat([u, dt, z, B.flatten(2), C.flatten(2)], -1), gpu)
        u, dt, z, B, C = packed.split([16, 16, 16, 8, 8], -1)
        rest = [t.to(gpu) for t in inputs]
        out = ops.selective_scan(u, dt, rest[2], B.unflatten(2, (1, 8)), C.unflatten(2, (1, 8)), rest[5], z, rest[7],
                                 state=rest[8])
        grad, = torch.autograd.grad(out, packed, back[0].to(gpu))
        with torch.no_grad():
            results, sizes = mixing.selective_scan(*map(fp64, inputs), [40, 40], True, fp64(back[0]), None)
        want = torch.cat([results[2], results[3], results[8], results[5].flatten(2), results[6].flatten(2)], -1)
        size = torch.cat([sizes[2], sizes[3], sizes[8], sizes[5].flatten(2), sizes[6].flatten(2)], -1)
        assert_close("packed", grad, want, size, 96 + 8 * 40 + 16)


@pytest.mark.parametrize("parts", [[1] * 7, [33, 40], [5, 1, 64, 1], [100, 100]])
def test_parts_of_a_sequence(gpu, parts):
    """A sequence in parts, each from the state that the part before left, is the whole."""
    inputs, _ = make(2, sum(parts), 40, 16, 1, FP32, seed=len(parts))
    there = [t.to(gpu) for t in inputs]
    with torch.no_grad():
        results, sizes = mixing.selective_scan(*map(fp64, inputs), [sum(parts)] * 2)
    kept, outs, at = there[8].clone(), [], 0
    for k in parts:
        v = [t[:, at:at + k] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(there)]
        v[8] = kept
        before = kept.clone()
        out, last = call([*v[:8], before], return_state=True)
        in_place = call(v, state_out=kept)
        assert torch.equal(out, in_place) and torch.equal(last, kept)
        outs.append(out)
        at += k
    assert_close("out", torch.cat(outs, 1), results[0], sizes[0], 96 + 8 * at)
    assert_close("state", kept, results[1], sizes[1], 96 + 8 * at)


@pytest.mark.parametrize("c,t,b", [(8, 4099, 1), (8, 300, 5), (512, 1100, 2), (512, 4200, 2)])
def test_chunks(gpu, c, t, b):
    """Few channels and many tokens: chunks side by side, with decays slow enough that states cross several.  Against the
    same call in parts that are one chunk each."""
    inputs, _ = make(b, t, c, 8, 1, FP32, seed=t)
    inputs[2] = inputs[2] * 0.02
    there = [x.to(gpu) for x in inputs]
    lengths = torch.tensor([t - 57 * i for i in range(b)], device=gpu)
    out, last = call(there, lengths, return_state=True)
    assert torch.equal(call(there, lengths), out)
    kept, outs = there[8].clone(), []
    for at in range(0, t, 64):  # two tiles: never more than one chunk
        v = [x[:, at:at + 64] if i in (0, 1, 3, 4, 6) else x for i, x in enumerate(there)]
        v[8] = kept
        outs.append(call(v, (lengths - at).clamp(0, 64), state_out=kept))
    # both are off by at most 8 roundings a token that a state lives for (0.02 * 0.1 * softplus(-2) a token: thousands)
    for a, w in ((out, torch.cat(outs, 1)), (last, kept)):
        assert (a - w).abs().max() <= 8 * t * 2.0 ** -24 * w.abs().max()


def test_long_gradient(gpu):
    """Many tiles: the carried gradient against the same pass in two parts, joined by the states' gradients."""
    inputs, back = make(1, 1500, 24, 16, 1, FP32)
    inputs[2] = inputs[2] * 0.05
    leaves = [leaf(t, gpu) for t in inputs]
    given = [t.to(gpu) for t in back]
    whole = torch.autograd.grad(call(leaves, return_state=True), leaves, given)
    head = [t[:, :701] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(leaves)]
    out, middle = call(head, return_state=True)
    tail = [t[:, 701:] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(leaves)]
    tail[8] = middle
    rest, last = call(tail, return_state=True)
    parts = torch.autograd.grad((torch.cat([out, rest], 1), last), leaves, given)
    for name, a, w in zip(NAMES[2:], whole, parts):
        # 8 roundings a token, and a rounding for each of the 1500 rows of a sum
        assert (a - w).abs().max() <= 9 * 1500 * 2.0 ** -24 * w.abs().max(), name


@pytest.mark.parametrize("which", range(9))
def test_one_gradient(gpu, which):
    """Each gradient alone, from one result alone, is the same bits as among all."""
    inputs, back = make(2, 70, 40, 16, 1, BF16)
    for result in (0, 1):
        if result == 1 and which in (4, 5, 6):
            continue  # the last state depends on none of C, D, z
        leaves = [leaf(t, gpu) for t in inputs]
        made = call(leaves, return_state=True)
        every = torch.autograd.grad(made[result], leaves, back[result].to(gpu), allow_unused=True)[which]
        leaves = [leaf(t, gpu) if i == which else t.to(gpu) for i, t in enumerate(inputs)]
        made = call(leaves, return_state=True)
        alone, = torch.autograd.grad(made[result], leaves[which], back[result].to(gpu))
        assert torch.equal(alone, every)


def test_no_tokens(gpu):
    for b, t in ((0, 4), (2, 0)):
        inputs, _ = make(b, t, 16, 8, 1, FP32)
        leaves = [leaf(x, gpu) for x in inputs]
        out, last = call(leaves, return_state=True)
        assert out.shape == (b, t, 16) and torch.equal(last, leaves[8])
        grads = torch.autograd.grad((out, last), leaves, (out.detach(), torch.ones_like(last)))
        assert all(not g.any() for g in grads[:8]) and torch.equal(grads[8], torch.ones_like(last))


def test_extremes(gpu):
    """Steps of nearly nothing and large ones, decays that underflow, growing states: what fp32 holds is held."""
    inputs, back = make(1, 12, 16, 8, 1, FP32, absent="b")
    inputs[1][0, 0], inputs[1][0, 1], inputs[1][0, 2] = -60.0, 30.0, -200.0
    inputs[1][0, 3:] = torch.linspace(-20, 6, 9)[:, None]
    inputs[2][:8] = -30.0
    inputs[2][8] = 0.5
    inputs[2][9] = 0.0
    leaves = [leaf(t, gpu) for t in inputs]
    made = call(leaves, return_state=True)
    grads = torch.autograd.grad(made, [t for t in leaves if t is not None], [t.to(gpu) for t in back])
    with torch.no_grad():
        results, sizes = mixing.selective_scan(*map(fp64, inputs), [12], True, *map(fp64, back))
    got = [*made, *grads]
    for name, a, w, size in zip([n for n in NAMES if n != "ddt_bias"], got, [w for w in results if w is not None],
                                [s for w, s in zip(results, sizes) if w is not None]):
        # an exponent of up to 30 * 30 is off by 2^-23 of itself where what is left is below exp(-900): a token of step 30
        # with decay 0.5 grows by exp(15), whose exponent 15 log2(e) = 22 is rounded twice: 44 roundings more a token
        assert_close(name, a, w, size, 96 + (8 + 44) * 12 + 16)


def test_differences(gpu):
    """The derivative along a direction from the results themselves, fp32: steps of 2^-7 leave 1e-4 of third derivatives
    and 2^-17 of rounding a value."""
    inputs, back = make(1, 6, 16, 8, 1, FP32, seed=5)
    there, given = [t.to(gpu) for t in inputs], [t.to(gpu) for t in back]
    leaves = [t.clone().requires_grad_() for t in there]
    grads = torch.autograd.grad(call(leaves, return_state=True), leaves, given)
    g = torch.Generator().manual_seed(9)

    def total(values):
        return sum((r.double() * b.double()).sum() for r, b in zip(call(values, return_state=True), given))

    for i, grad in enumerate(grads):
        step, h = randn(g, *there[i].shape).to(gpu), 2.0 ** -7
        ends = [total([t + s * h * step if j == i else t for j, t in enumerate(there)]) for s in (1, -1)]
        want = (ends[0] - ends[1]) / (2 * h)
        scale = (grad.double() * step).abs().sum() + 10
        assert abs((grad.double() * step).sum() - want) <= 2e-3 * scale, i


def test_growing_states(gpu):
    """Decays above one: a state that is zero stays so, and a small one is finite where the power of a whole chunk is not."""
    b, t, c, n = 1, 400, 8, 8
    zeros = torch.zeros(b, t, c, device=gpu)
    dt, A = torch.full((b, t, c), 1.0, device=gpu), torch.full((c, n), 0.5, device=gpu)  # exp(200) over the call
    maps = torch.ones(b, t, 1, n, device=gpu)
    out, last = ops.selective_scan(zeros, dt, A, maps, maps, softplus=False, return_state=True)
    assert not out.any() and not last.any()
    first = torch.full((b, c, n), 1e-37, device=gpu)
    out, last = ops.selective_scan(zeros[:, :340], dt[:, :340], A, maps[:, :340], maps[:, :340], state=first, softplus=False,
                                   return_state=True)
    want = 1e-37 * torch.exp(torch.tensor(170.0, dtype=torch.float64))  # 6.6e36
    # 340 decays of 2 roundings and 2 of their exponent, as many products
    assert (last.double().cpu() - want).abs().max() <= 5 * 340 * 2.0 ** -24 * want
    leaves = [zeros.clone().requires_grad_(), first.clone().requires_grad_()]
    out = ops.selective_scan(leaves[0], dt, A, maps, maps, state=leaves[1], softplus=False)
    du, ds = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert not du.any() and not ds.any()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_state_in_place(gpu, mode):
    """A decoder's state, made inside or outside the mode, moves on in place; writing over a leaf is refused."""
    inputs, _ = make(2, 3, 16, 8, 1, FP32)
    outside = [x.to(gpu) for x in inputs]
    with mode():
        inside = [x.to(gpu) for x in inputs]
        for v in (outside, inside):
            want = call(v, return_state=True)[1].clone()
            call(v, state_out=v[8])
            assert torch.equal(v[8], want)
    fresh = outside[8].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="return_state"):
        call([*outside[:8], None], state_out=fresh)
    with pytest.raises(RuntimeError, match="return_state"):
        call([x.requires_grad_() if i == 0 else x for i, x in enumerate(outside)], state_out=outside[8].clone())
