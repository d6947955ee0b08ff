"""The sequence mixing operators where offsets pass 32 bits: more than 2^31 elements, and token strides near 2^25.

The ends of a large call against the same rows in a small one.  The frame and the convolution work row by row: the same
bits.  The scan's small call is cut into tiles and chunks elsewhere: its states forget 192 tokens wholly (a step of at
least log(1 + e^0.5) = 0.97 and A <= -1: exp(-186)), and what is compared is off by 96 + 8 x 192 roundings of 2^-24 on
either side, 2e-4 of the largest value, and by the rounding to bf16 of both, a step (eps) of the value."""

import pytest
import torch

from boltz_lumi_amd import ops
from mixing_cases import BF16, FP32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def randn(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device=g.device, dtype=dtype)


def test_residual_norm(gpu):
    g = torch.Generator(gpu).manual_seed(0)
    t, d = 262_147, 8192
    x, y, gate, dr, dh = (randn(g, 1, t, d) for _ in range(5))
    weights = [randn(g, d) for _ in range(3)]

    def run(*rows):
        leaves = [v.detach().requires_grad_() for v in rows[:3]]
        r, h = ops.residual_norm(*leaves, *weights)
        return [r.detach(), h.detach(), *torch.autograd.grad((r, h), leaves, rows[3:])]

    whole = run(x, y, gate, dr, dh)
    for part in (slice(0, 70), slice(t - 70, t)):
        small = run(*(v[:, part].contiguous() for v in (x, y, gate, dr, dh)))
        assert all(torch.equal(a[:, part], b) for a, b in zip(whole, small))


def test_causal_conv(gpu):
    g = torch.Generator(gpu).manual_seed(1)
    t, c = 131_083, 16_384
    x, dy = randn(g, 1, t, c), randn(g, 1, t, c)
    w, b = randn(g, c, 4), randn(g, c)

    def run(x, dy):
        x = x.detach().requires_grad_()
        y, last = ops.causal_conv(x, w, b, return_state=True)
        return [y.detach(), *torch.autograd.grad((y, last), x, (dy, torch.ones_like(last))), last.detach()]

    whole = run(x, dy)
    with torch.no_grad():
        assert torch.equal(ops.causal_conv(x[:, :64], w, b), whole[0][:, :64])
    small = run(x[:, -103:].contiguous(), dy[:, -103:].contiguous())
    for a, s in zip(whole[:2], small[:2]):
        assert torch.equal(a[:, -100:], s[:, 3:])
    assert torch.equal(whole[2], small[2])


def near(name, a, w):
    a, w = a.float(), w.float()
    limit = torch.finfo(BF16).eps * torch.maximum(a.abs(), w.abs()) + 2e-4 * w.abs().max()
    assert torch.isfinite(a).all() and ((a - w).abs() <= limit).all(), (name, ((a - w).abs() / limit).max())


def test_selective_scan(gpu):
    g = torch.Generator(gpu).manual_seed(2)
    t, c, n = 131_083, 16_384, 8
    u, z, dout = (randn(g, 1, t, c) for _ in range(3))
    dt = torch.rand(1, t, c, generator=g, device=gpu, dtype=BF16) + 0.5
    B, C = (randn(g, 1, t, 1, n) for _ in range(2))
    A, D = -1 - torch.rand(c, n, generator=g, device=gpu), randn(g, c, dtype=FP32)

    def run(u, dt, B, C, z, dout):
        leaves = [v.detach().requires_grad_() for v in (u, dt, B, C, z)]
        out = ops.selective_scan(leaves[0], leaves[1], A, leaves[2], leaves[3], D, leaves[4])
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    tensors = u, dt, B, C, z, dout
    whole = run(*tensors)
    for part, compared in ((slice(0, 256), slice(0, 64)), (slice(t - 256, t), slice(192, 256))):
        small = run(*(v[:, part].contiguous() for v in tensors))
        for name, a, w in zip(("out", "du", "ddt", "dB", "dC", "dz"), whole, small):
            near(name, a[:, part][:, compared], w[:, compared])


@pytest.mark.parametrize("stride", [(1 << 25) - 4, 1 << 25])
@pytest.mark.parametrize("n", [8, 64])
def test_selective_scan_strides(gpu, stride, n):
    """One projection, 33 tokens, its rows as far apart as they may be and a step further (copied): the same bits."""
    g = torch.Generator(gpu).manual_seed(3)
    t, c = 33, 24
    rows = torch.empty(1, t, stride, device=gpu, dtype=FP32)
    rows[:, :, :3 * c + 2 * n] = randn(g, 1, t, 3 * c + 2 * n, dtype=FP32)
    u, dt, z, B, C = rows[:, :, :3 * c + 2 * n].split([c, c, c, n, n], -1)
    B, C = B[:, :, None], C[:, :, None]
    A = -torch.rand(c, n, generator=g, device=gpu)

    def run(*tensors):
        leaves = [v.detach().requires_grad_() for v in tensors]
        out = ops.selective_scan(leaves[0], leaves[1], A, leaves[2], leaves[3], z=leaves[4])
        return [out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))]

    far, dense = run(u, dt, B, C, z), run(*(v.contiguous() for v in (u, dt, B, C, z)))
    assert all(torch.equal(a, b) for a, b in zip(far, dense))
