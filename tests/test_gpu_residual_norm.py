"""ops.residual_norm and its gradients against the oracle in fp64.

Tolerances: half a step of the result's type, and 64 roundings of 2^-24 relative to the magnitudes that a value is made
of: the sums of squares (a thread's 8 V values in a row, then at most ten pairwise levels: under 32), their root and
reciprocal, a sigmoid of the hardware exponential and reciprocal (4), the products.  Sums over rows add one per row."""

import pytest
import torch

from boltz_lumi_amd import ops
from oracle import mixing
from mixing_cases import BF16, FP32, assert_close, fp64, leaf, randn

pytestmark = pytest.mark.gpu

NAMES = ["r", "h", "dx", "dy", "dgate", "dy_weight", "dscale", "dweight"]


def make(b, t, d, stream, dtype, gate, weights, w_dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x, y = randn(g, b, t, d, dtype=stream, scale=2.0), randn(g, b, t, d, dtype=dtype)
    gates = {"none": None, "token": (b, t, d), "sample": (b, 1, d)}[gate]
    gates = None if gates is None else randn(g, *gates, dtype=dtype)
    yw, k, w = (randn(g, d, dtype=w_dtype, scale=0.3, shift=1.0) if c in weights else None for c in "ykw")
    return [x, y, gates, yw, k, w], [randn(g, b, t, d, dtype=stream), randn(g, b, t, d, dtype=dtype)]


def check(inputs, back, gpu, post=True, pre=True, eps=1e-6, view=lambda t: t):
    leaves = [leaf(t, gpu) for t in inputs]
    seen = [None if t is None else view(t) if t.dim() == 3 else t for t in leaves]
    made = ops.residual_norm(*seen, eps=eps, post_norm=post, pre_norm=pre)
    made = made if pre else (made,)
    given = [t.to(gpu) for t in back[:len(made)]]
    wanted = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(made, wanted, given))
    got = [*made, *(None if t is None else next(grads) for t in leaves)]
    with torch.no_grad():
        results, sizes = mixing.residual_norm(*map(fp64, inputs), eps, *map(fp64, back), post_norm=post, pre_norm=pre)
    rows = inputs[0].shape[0] * inputs[0].shape[1]
    names = NAMES if pre else [NAMES[0], *NAMES[2:]]
    for name, a, b, size in zip(names, got, results, sizes):
        if a is not None and b is not None:
            assert_close(name, a, b, size, 64 + (rows if name[0] == "d" and name not in ("dx", "dy") else 0))
    return got


@pytest.mark.parametrize("d", [8, 24, 120, 128, 136, 384, 512, 520, 768, 1024, 1032, 1536, 2048, 2056, 4096, 4104, 8192])
def test_widths(gpu, d):
    check(*make(2, 5, d, FP32, BF16, "token", "ykw", FP32, seed=d), gpu)


@pytest.mark.parametrize("stream,dtype,w_dtype", [(FP32, FP32, FP32), (FP32, BF16, BF16), (BF16, BF16, BF16),
                                                  (BF16, BF16, FP32)])
@pytest.mark.parametrize("gate", ["none", "token", "sample"])
def test_types_and_gates(gpu, stream, dtype, w_dtype, gate):
    check(*make(3, 37, 200, stream, dtype, gate, "ykw", w_dtype), gpu)
    check(*make(2, 3, 1200, stream, dtype, gate, "ykw", w_dtype), gpu)


@pytest.mark.parametrize("b,t", [(1, 1), (32, 1), (1, 700), (3, 129), (600, 2), (1, 5000)])
@pytest.mark.parametrize("gate", ["token", "sample"])
def test_rows(gpu, b, t, gate):
    check(*make(b, t, 64, BF16, BF16, gate, "ykw", FP32), gpu)


@pytest.mark.parametrize("weights", ["", "y", "k", "w", "yw"])
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False), (False, False)])
def test_absent_parts(gpu, weights, post, pre):
    kept = "".join(c for c in weights if not (c == "y" and not post) and not (c == "w" and not pre))
    check(*make(2, 9, 136, FP32, FP32, "token", kept, FP32), gpu, post, pre)


def test_strides(gpu):
    """Column slices, transposed batches, expanded gates and layouts that have to be copied."""
    inputs, back = make(3, 7, 96, BF16, BF16, "token", "ykw", FP32)

    def slices(t):
        wide = torch.full((t.shape[0], t.shape[1], 3 * t.shape[2]), float("nan"), device=t.device, dtype=t.dtype)
        wide[..., 96:192] = t
        return wide[..., 96:192]

    for view in (slices, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)):
        check(inputs, back, gpu, view=view)
    gate = randn(torch.Generator().manual_seed(3), 1, 1, 96, dtype=BF16)
    leaves = [leaf(t, gpu) for t in (inputs[0], inputs[1], gate, *inputs[3:])]
    made = ops.residual_norm(leaves[0], leaves[1], leaves[2].expand(3, 1, 96), *leaves[3:])
    dgate, = torch.autograd.grad(made, leaves[2], [t.to(gpu) for t in back])
    with torch.no_grad():
        results, sizes = mixing.residual_norm(*map(fp64, (inputs[0], inputs[1], gate.expand(3, 1, 96), *inputs[3:])), 1e-6,
                                              *map(fp64, back))
    # torch adds the three elements' gradients, each rounded to bf16: a half step each
    size = sizes[4].sum(0, keepdim=True) + 2.0 ** 15 * results[4].abs().sum(0, keepdim=True)
    assert_close("dgate", dgate, results[4].sum(0, keepdim=True), size, 64 + 21)


@pytest.mark.parametrize("which", range(6))
def test_one_gradient(gpu, which):
    """Each gradient alone, from one result alone, is the same bits as among all."""
    inputs, back = make(2, 33, 264, FP32, BF16, "sample", "ykw", FP32)
    for result in (0, 1):
        leaves = [leaf(t, gpu) for t in inputs]
        made = ops.residual_norm(*leaves)
        if which == 5 and result == 0:
            continue  # r does not depend on the next norm's weight
        every = torch.autograd.grad(made[result], leaves, back[result].to(gpu), allow_unused=True)[which]
        leaves = [t.to(gpu) if i != which else leaf(t, gpu) for i, t in enumerate(inputs)]
        alone, = torch.autograd.grad(ops.residual_norm(*leaves)[result], leaves[which], back[result].to(gpu))
        assert torch.equal(alone, every)


def test_same_bits_with_and_without_gradients(gpu):
    inputs, _ = make(2, 300, 768, FP32, BF16, "token", "ykw", FP32)
    there = [t.to(gpu) for t in inputs]
    with torch.no_grad():
        plain = ops.residual_norm(*there)
    taped = ops.residual_norm(*[t.requires_grad_() for t in there])
    assert all(torch.equal(a, b) for a, b in zip(plain, taped))


def test_no_rows(gpu):
    for b, t in ((0, 4), (2, 0)):
        inputs, _ = make(b, t, 16, FP32, FP32, "token", "ykw", FP32)
        leaves = [leaf(x, gpu) for x in inputs]
        r, h = ops.residual_norm(*leaves)
        assert r.shape == h.shape == (b, t, 16)
        grads = torch.autograd.grad((r, h), leaves, (r.detach(), h.detach()))
        assert all(not g.any() and g.shape == x.shape for g, x in zip(grads, leaves))


def test_zero_rows_and_extremes(gpu):
    """Rows of zeros (the norm's eps alone), tiny and large values, saturated gates."""
    inputs, back = make(1, 8, 64, FP32, FP32, "token", "ykw", FP32)
    x, y, gate = inputs[:3]
    x[0, 0] = y[0, 0] = 0
    y[0, 1] = 0
    x[0, 2], y[0, 2] = x[0, 2] * 1e-3, y[0, 2] * 1e-4
    x[0, 3], y[0, 3] = x[0, 3] * 1e6, y[0, 3] * 1e8
    gate[0, 4], gate[0, 5] = 40.0, -40.0
    gate[0, 6] = torch.where(torch.arange(64) % 2 == 0, 1e30, -1e30)
    check(inputs, back, gpu)


def test_differences(gpu):
    """The derivative along a direction from the results themselves, fp32: a difference of step h is off by h^2 times
    third derivatives (about 1 a value here) and by 2^-24 / h a value; h = 2^-7 leaves 1e-4."""
    inputs, back = make(2, 6, 64, FP32, FP32, "sample", "ykw", FP32, seed=5)
    there, given = [t.to(gpu) for t in inputs], [t.to(gpu) for t in back]
    g = torch.Generator().manual_seed(9)

    def total(values):
        return sum((r.double() * b.double()).sum() for r, b in zip(ops.residual_norm(*values), given))

    leaves = [t.clone().requires_grad_() for t in there]
    grads = torch.autograd.grad(ops.residual_norm(*leaves), leaves, given)
    for i, grad in enumerate(grads):
        step = randn(g, *there[i].shape).to(gpu)
        h = 2.0 ** -7
        moved = [total([t + s * h * step if j == i else t for j, t in enumerate(there)]) for s in (1, -1)]
        want = (moved[0] - moved[1]) / (2 * h)
        scale = (grad.double() * step).abs().sum() + 10
        assert abs((grad.double() * step).sum() - want) <= 2e-3 * scale, i


@pytest.mark.parametrize("eps", [0.0, -1e-6, 2.0 ** -127, float("nan")])
def test_eps_is_refused(gpu, eps):
    x = torch.ones(1, 2, 8, device=gpu)
    with pytest.raises(RuntimeError, match="eps"):
        ops.residual_norm(x, x, eps=eps)
