"""Cross attention whose logits lie far from zero: masks written as a bias of a
large finite value, and large logits without a bias, forward and all gradients
against 64 bits.

Queries and keys are small whole numbers (times a power of two) and the scale is
a power of two where a bias is added, so every product is exact in 32 bits and a
logit is rounded once, by the addition of the bias: the reference rounds it there too
(at 1e9 an fp32 logit is a multiple of 64) and takes the rest in 64 bits.

Tolerances are those of test_gpu_cross_attention.check: a result is within 2^-14 of the
sum of its terms' magnitudes (large bf16 calls: and half a step, 2^-8, of it for their weights), and half
a step of itself. The 2^-14 is made of a weight's exponent (rounded once or twice, 2^-24 of at
most 126 where the weight is not zero, and at most 2^-16.5 for a reference point below 2^8), its 16 bits in
bf16 (2^-16), and sums of at most 520 terms in a chain (2^-15, if every rounding went one way). dP and
delta are sums of up to 64 products, and bf16 takes delta from an output of 16 bits: their difference is
within 2^-16 of the products' magnitudes, which do not vanish where dP does (rows of a single
weight, whose dP - delta is zero), so a fourth of those is added to the magnitudes that the 2^-14 multiplies.

Large bf16 calls divide by the sum of their rounded weights w (1 + d_i), |d_i| <= 2^-8. In the forward
pass those are the weights used, and a row's dominant one is divided by its own rounding. The gradients compute
P = w / sum w (1 + d_i) anew, off by up to 2^-8 where one weight dominates (its sum's error is its own), and
round it or dS once more, 2^-8: twice 2^-8 of the terms in all, so twice the sizes."""

import pytest
import torch
from test_gpu_cross_attention import check

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu


def formula(x, q, k, v, scale, dout):
    """(out, dq, dk, dv, dx) from the logits x [B, H, M, N] (exact, fp64), beside each the sum of its terms' magnitudes."""
    h, hk = q.shape[2], k.shape[2]
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, dout))
    k, v = (t.repeat_interleave(h // hk, 1) for t in (k, v))
    p = x.softmax(-1)
    out = torch.matmul(p, v)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (do * out).sum(-1, keepdim=True))
    terms = dp.abs() + torch.matmul(do.abs(), v.abs().transpose(2, 3)) / 4
    size = p * (terms + (p * terms).sum(-1, keepdim=True))

    def rows(t):
        return t.transpose(1, 2)

    def keys(t):
        return t.unflatten(1, (hk, h // hk)).sum(2).transpose(1, 2)

    return {"out": (rows(out), rows(torch.matmul(p, v.abs()))),
            "dq": [rows(torch.matmul(a, b)) * scale for a, b in ((ds, k), (size, k.abs()))],
            "dk": [keys(torch.matmul(a.transpose(2, 3), b)) * scale for a, b in ((ds, q), (size, q.abs()))],
            "dv": [keys(torch.matmul(p.transpose(2, 3), b)) for b in (do, do.abs())],
            "dbias": (ds, size)}


def compare(got, want, large):
    for (name, (ref, size)), have in zip(want.items(), got):
        assert torch.isfinite(have).all(), name
        check(have, ref, size * 2 if large and name != "out" else size, name, weights=large)


def whole(g, *shape, dtype):
    return torch.randint(-2, 3, shape, generator=g, device=g.device).to(dtype)


def patterns(n, device):
    """Keys that carry the large value: all, the first tile, half a call (a split or more), one wave's keys of a decoding
    step, all but the last ones (left padding), every other one, the last half, none."""
    j = torch.arange(n, device=device)
    return torch.stack([j >= 0, j < 32, j < n // 2, j // 32 % 4 == 1, j < n - 3, j % 2 == 0, j >= n // 2, j < 0])


SHAPES = [  # batch, m, n, heads, kv_heads, dim
    (2, 1, 300, 16, 2, 64),  # a decoding step
    (1, 2, 4200, 8, 1, 64),  # and one whose keys are split
    (2, 20, 150, 2, 2, 32),
    (2, 70, 300, 4, 2, 64),
    (1, 40, 2200, 2, 1, 64),  # split
    (1, 520, 1031, 8, 4, 64),  # bf16 weights of 8 bits
]
LARGE = SHAPES[-1]
VALUES = [-1e4, -1e6, -1e8, -4e8, -1e9, -1e10, -1e30, -9e37, -3.3e38, 1e6, 3e8, 1e9, 1e30]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("value", VALUES)
def test_large_finite_bias(gpu, dtype, shape, value):
    print(f"bias of {value} {shape} {dtype}", flush=True)
    b, m, n, h, hk, d = shape
    g = torch.Generator(device=gpu).manual_seed(m + n)
    q, k = whole(g, b, m, h, d, dtype=dtype), whole(g, b, n, hk, d, dtype=dtype)
    v, dout = (torch.randn(b, t, x, d, generator=g, device=gpu).to(dtype) for t, x in ((n, hk), (m, h)))
    pick = (torch.arange(h, device=gpu)[:, None] + torch.arange(m, device=gpu)) % 8
    bias = torch.where(patterns(n, gpu)[pick], value, whole(g, h, m, n, dtype=torch.float32) / 4).to(dtype)[None]
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    out = ops.cross_attention(q, k, v, bias=bias, scale=0.125)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        again = ops.cross_attention(q, k, v, bias=bias, scale=0.125)
        s = torch.matmul(q.double().transpose(1, 2), k.double().permute(0, 2, 3, 1).repeat_interleave(h // hk, 1))
        x = (s * 0.125 + bias.double()).float().double()
        want = formula(x, q, k, v, 0.125, dout)
    assert torch.equal(out.detach(), again)
    want["dbias"] = [t.sum(0, keepdim=True) for t in want["dbias"]]
    compare((out.detach(), *grads), want, shape == LARGE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("power,scale", [(4, 0.125), (7, 0.1), (13, 0.1), (20, 0.1), (30, 0.125), (34, 0.1), (60, 0.1),
                                         (100, 0.125)])
def test_large_logits(gpu, dtype, shape, power, scale):
    """No bias: the logits are scale * 2^power * whole numbers, with ties. Queries are negated in half of the heads' rows."""
    print(f"logits of 2^{power} {scale} {shape} {dtype}", flush=True)
    b, m, n, h, hk, d = shape
    g = torch.Generator(device=gpu).manual_seed(m + n)
    q, k = whole(g, b, m, h, d, dtype=dtype), whole(g, b, n, hk, d, dtype=dtype)
    k[..., :d // 2] = 2  # whole rows of large logits of one sign
    turn = (torch.arange(m, device=gpu)[:, None, None] + torch.arange(h, device=gpu)[:, None]) % 2
    q = q.abs() * (1 - 2 * turn).to(dtype)
    q = (q * 2.0 ** power).to(dtype)
    v, dout = (torch.randn(b, t, x, d, generator=g, device=gpu).to(dtype) for t, x in ((n, hk), (m, h)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(q, k, v, scale=scale)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        scale = torch.tensor(scale, dtype=torch.float32).item()  # as the kernels take it
        s = torch.matmul(q.double().transpose(1, 2), k.double().permute(0, 2, 3, 1).repeat_interleave(h // hk, 1))
        want = formula(s * scale, q, k, v, scale, dout)
    compare((out.detach(), *grads), want, shape == LARGE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_minus_infinity(gpu, dtype, shape):
    """-inf over the same patterns: whole rows give zeros and zero gradients, whatever tiles, waves or splits hold one."""
    print(f"bias of -inf {shape} {dtype}", flush=True)
    b, m, n, h, hk, d = shape
    g = torch.Generator(device=gpu).manual_seed(m + n)
    q, k = whole(g, b, m, h, d, dtype=dtype), whole(g, b, n, hk, d, dtype=dtype)
    v, dout = (torch.randn(b, t, x, d, generator=g, device=gpu).to(dtype) for t, x in ((n, hk), (m, h)))
    pick = (torch.arange(h, device=gpu)[:, None] + torch.arange(m, device=gpu)) % 8
    bias = torch.where(patterns(n, gpu)[pick], -torch.inf, whole(g, h, m, n, dtype=torch.float32) / 4).to(dtype)[None]
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    out = ops.cross_attention(q, k, v, bias=bias, scale=0.125)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        s = torch.matmul(q.double().transpose(1, 2), k.double().permute(0, 2, 3, 1).repeat_interleave(h // hk, 1))
        x = s * 0.125 + bias.double()
        empty = (x == -torch.inf).all(-1, keepdim=True)
        want = formula(torch.where(empty, 0.0, x), q, k, v, 0.125, torch.where(empty.transpose(1, 2), 0.0, dout))
        want["out"] = [torch.where(empty.transpose(1, 2), 0.0, t) for t in want["out"]]
    want["dbias"] = [t.sum(0, keepdim=True) for t in want["dbias"]]
    compare((out.detach(), *grads), want, shape == LARGE)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("form", [(0, 1), (1, 1), (1, 0)])  # of the bias: per batch element, per head
def test_a_left_out_keys_bias_is_never_looked_at(gpu, dtype, shape, form):
    print(f"bias of left-out keys {shape} {form} {dtype}", flush=True)
    b, m, n, h, hk, d = shape
    g = torch.Generator(device=gpu).manual_seed(m + n)
    q, k, v = (torch.randn(b, t, x, d, generator=g, device=gpu).to(dtype) for t, x in ((m, h), (n, hk), (n, hk)))
    mask = torch.rand(b, n, generator=g, device=gpu) < 0.6
    mask[:, :40] = False
    mask[-1] &= b == 1
    both = mask if form[0] else mask.any(0, keepdim=True)  # keys of some element that shares the bias
    bias = torch.randn(b if form[0] else 1, h if form[1] else 1, m, n, generator=g, device=gpu).to(dtype)
    dout = torch.randn(b, m, h, d, generator=g, device=gpu).to(dtype)

    def run(bias):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, bias)]
        out = ops.cross_attention(*leaves[:3], mask, leaves[3])
        return out.detach(), *torch.autograd.grad(out, leaves, dout)

    clean = run(bias)
    for value in (torch.nan, torch.inf, torch.finfo(dtype).min):
        dirty = run(torch.where(both[:, None, None], bias, value))
        assert all(torch.equal(x, y) for x, y in zip(clean, dirty)), value
    assert torch.isfinite(clean[-1]).all() and not clean[-1].masked_select(~both[:, None, None]).any()
