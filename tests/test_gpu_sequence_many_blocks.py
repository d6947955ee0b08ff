"""Calls of more blocks than a launch takes along one axis (2^32 threads, so 2^24 blocks of 256): many small batch
elements, or very many rows.  A sample of the elements on both sides of every border of the grid against
64 bits, tolerances as in test_gpu_cross_attention_far: with two or three keys a row often has one weight, where dP and
delta cancel and their difference is bounded by 2^-16 of their products' magnitudes (delta is taken from an output of
16 bits), not of dP."""

import pytest
import torch
from test_gpu_cross_attention import check, randn
from test_gpu_cross_attention_far import compare, formula

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu


def sample(count, g):
    """Indices below count: the ends, the middle (where a folded grid's second row starts) and some others."""
    ends = [torch.arange(40), torch.arange(count // 2 - 40, count // 2 + 40), torch.arange(count - 40, count)]
    return torch.cat([*(t.to(g.device) for t in ends), torch.randint(0, count, (300,), generator=g, device=g.device)])


def logits(q, k, bias, scale):
    k = k.double().permute(0, 2, 3, 1).repeat_interleave(q.shape[2] // k.shape[2], 1)
    s = torch.matmul(q.double().transpose(1, 2), k.contiguous()) * scale
    return s if bias is None else s + bias.double()


def test_attention_of_many_elements(gpu):
    """Every kernel of a decoding-sized call, with a bias that the heads share (its gradient has a kernel of its own)."""
    b, m, n, h, hk, d = (1 << 24) + 9, 1, 2, 2, 1, 8
    g = torch.Generator(device=gpu).manual_seed(0)
    q, k, v, dout = (randn(g, b, t, x, d, dtype=torch.bfloat16) for t, x in ((m, h), (n, hk), (n, hk), (m, h)))
    bias = randn(g, b, 1, m, n, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    out = ops.cross_attention(q, k, v, bias=bias)
    grads = torch.autograd.grad(out, leaves, dout)
    at = sample(b, g)
    with torch.no_grad():
        x = logits(q[at], k[at], bias[at], d ** -0.5)
        want = formula(x, q[at], k[at], v[at], d ** -0.5, dout[at])
        want["dbias"] = [t.sum(1, keepdim=True) for t in want["dbias"]]
        compare([t[at] for t in (out.detach(), *grads)], want, False)


def test_attention_of_many_rows(gpu):
    """The row sums of the gradients take a block for sixteen rows: 2^28 rows and a few."""
    b, m, n, h, hk, d = 1, (1 << 27) + 5, 3, 2, 2, 8
    g = torch.Generator(device=gpu).manual_seed(1)
    k, v = (randn(g, b, n, hk, d, dtype=torch.bfloat16) for _ in range(2))
    pattern = randn(g, b, 1 << 10, h, d, dtype=torch.bfloat16)
    q = pattern.repeat(1, m // pattern.shape[1] + 1, 1, 1)[:, :m].requires_grad_()
    out = ops.cross_attention(q, k, v)
    dq, = torch.autograd.grad(out, q, out.detach())
    at = sample(m, g)
    with torch.no_grad():
        want = formula(logits(q[:, at], k, None, d ** -0.5), q[:, at], k, v, d ** -0.5, out[:, at])
        check(out[:, at], *want["out"], "out", weights=False)
        check(dq[:, at], *want["dq"], "dq", weights=False)


def test_table_gradient_of_many_planes(gpu):
    batch, heads = (1 << 20) + 3, 16
    g = torch.Generator(device=gpu).manual_seed(2)
    table = torch.randn(4, heads, generator=g, device=gpu, requires_grad=True)
    q_pos, k_pos = (torch.randint(0, 5, (batch, 1), generator=g, device=gpu) for _ in range(2))
    bias = ops.relative_bias(table, q_pos, k_pos, exact=1, max_distance=3)
    dbias = torch.randint(-8, 9, bias.shape, generator=g, device=gpu).float()  # sums of whole numbers are exact
    dtable, = torch.autograd.grad(bias, table, dbias)
    d = (k_pos - q_pos)[:, 0]
    bucket = (d.abs() >= 1).long() + 2 * (d > 0)
    want = torch.stack([dbias[bucket == c].sum(0, dtype=torch.float64).flatten() for c in range(4)])
    assert torch.equal(dtable.double(), want)
