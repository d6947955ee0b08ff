"""The sequence operators together, as a decoder block uses them: query / key
norm with rotation and a relative bias feed self attention, another norm feeds
attention to an encoder's padded states; values and gradients of the chain
against 64 bits, the chain captured in a graph, a decoding step against the
whole sequence, and the relative bias in the framework's own pair-biased
attention.

Tolerance of the chain, fp32: each operator is within 2^-14 of the sum of its
terms' magnitudes (their own tests); three in a row, whose sums stay within a
factor of four of their results' maxima here, are within 2^-10 of the largest
value of each result."""

import math

import pytest
import torch

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu

B, M, N, H, HK, D = 2, 45, 83, 8, 2, 32
EPS = 1e-6


def make(gpu, dtype, grad):
    g = torch.Generator(device=gpu).manual_seed(0)

    def randn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=gpu) * scale + shift).to(dtype)

    x = {"q": randn(B, M, H, D), "k": randn(B, M, HK, D), "v": randn(B, M, HK, D), "xk": randn(B, N, HK, D),
         "xv": randn(B, N, HK, D), "qw": randn(D, scale=0.1, shift=1), "kw": randn(D, scale=0.1, shift=1),
         "table": randn(32, H)}
    leaves = {name: t.requires_grad_(grad) for name, t in x.items()}
    pos, xpos = torch.arange(M, device=gpu), torch.arange(N, device=gpu)
    inv = 10000.0 ** (-torch.arange(D // 2, device=gpu, dtype=torch.float64) / (D // 2))
    mask = torch.arange(N, device=gpu) < torch.tensor([N, N // 3], device=gpu)[:, None]
    return leaves, (pos, xpos, inv, mask)


def chain(x, consts):
    pos, xpos, inv, mask = consts
    q, k = ops.qk_norm_rope(x["q"], x["k"], x["qw"], x["kw"], pos, pos, inv, eps=EPS)
    bias = ops.relative_bias(x["table"], pos, pos, exact=8, max_distance=40)
    y = ops.cross_attention(q, k, x["v"], bias=bias[None])
    q, k = ops.qk_norm_rope(y, x["xk"], x["qw"], x["kw"], pos, xpos, inv, eps=EPS)
    return ops.cross_attention(q, k, x["xv"], mask=mask)


def plain_chain(x, consts):
    pos, xpos, inv, mask = consts

    def norm_rope(t, w, p):
        n = t / (t.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        angle = (p.double()[:, None] * inv)[:, None]
        a, b = n.chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1)

    def attention(q, k, v, bias, mask):
        k, v = (t.repeat_interleave(H // HK, 2) for t in (k, v))
        s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * D ** -0.5
        s = s if bias is None else s + bias
        s = s if mask is None else s.masked_fill(~mask[:, None, None], -math.inf)
        return torch.matmul(s.softmax(-1), v.transpose(1, 2)).transpose(1, 2)

    edges = torch.tensor(list(ops._relative_thresholds(16, 8, 40)), device=pos.device)
    d = pos[None, :] - pos[:, None]
    bucket = torch.bucketize(d.abs(), edges, right=True) + 16 * (d > 0)
    bias = x["table"][bucket].movedim(-1, 0)
    y = attention(norm_rope(x["q"], x["qw"], pos), norm_rope(x["k"], x["kw"], pos), x["v"], bias, None)
    return attention(norm_rope(y, x["qw"], pos), norm_rope(x["xk"], x["kw"], xpos), x["xv"], None, mask)


def test_chain_against_64_bits(gpu):
    x, consts = make(gpu, torch.float32, True)
    out = chain(x, consts)
    dout = torch.randn_like(out)
    grads = torch.autograd.grad(out, list(x.values()), dout)
    x64 = {name: t.detach().double().requires_grad_() for name, t in x.items()}
    want = plain_chain(x64, consts)
    want_grads = torch.autograd.grad(want, list(x64.values()), dout.double())
    for name, got, ref in zip(("out", *x), (out.detach(), *grads), (want.detach(), *want_grads)):
        err = (got.double() - ref).abs().max().item()
        assert err <= 2.0 ** -10 * ref.abs().max().item(), (name, err)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chain_captured(gpu, dtype):
    """Forward and backward in one graph, replayed with eager work between: the same bits as eager each time."""
    x, consts = make(gpu, dtype, False)
    dout = torch.randn(B, M, H, D, device=gpu).to(dtype)

    def once():
        leaves = {name: t.detach().requires_grad_() for name, t in x.items()}
        out = chain(leaves, consts)
        return out.detach(), *torch.autograd.grad(out, list(leaves.values()), dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for step in (0.0, 0.25, -0.5):
        for name in ("q", "xk", "table"):
            x[name].add_(step)
        want = once()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_decoding_step_is_the_last_row(gpu):
    """A new token alone (few rows, split keys) against the whole sequence's last row: the same formula in another
    order, so within twice the operator's fp32 bound of the row's largest value."""
    x, (pos, xpos, inv, mask) = make(gpu, torch.float32, False)
    with torch.no_grad():
        q, k = ops.qk_norm_rope(x["q"], x["k"], x["qw"], x["kw"], pos, pos, inv)
        one, _ = ops.qk_norm_rope(x["q"][:, -1:], None, x["qw"], None, pos[-1:], None, inv)
        assert torch.equal(one, q[:, -1:])
        bias = ops.relative_bias(x["table"], pos, pos)
        row = ops.relative_bias(x["table"], pos[-1:], pos)
        assert torch.equal(row, bias[:, -1:])
        whole = ops.cross_attention(q, k, x["v"], bias=bias[None])[:, -1:]
        last = ops.cross_attention(one, k, x["v"], bias=row[None])
        assert (last - whole).abs().max().item() <= 2.0 ** -13 * x["v"].abs().max().item()


def test_relative_bias_in_the_pair_biased_attention(gpu):
    """bias [1, H, N, N] as ops.seq_attention_batched takes it, against cross_attention with the same bias: two
    kernels for one formula, fp32 both."""
    g = torch.Generator(device=gpu).manual_seed(1)
    n, heads, d = 77, 16, 24
    q, k, v = (torch.randn(3, n, heads * d, generator=g, device=gpu) for _ in range(3))
    table, pos = torch.randn(66, heads, generator=g, device=gpu), torch.arange(n, device=gpu)
    with torch.inference_mode():
        bias = ops.relative_bias(table, pos, pos, exact=32)[None]
        far = torch.full_like(q, 100.0)  # the gate's sigmoid is 1
        mask = torch.arange(n, device=gpu) < n - 3
        own = ops.seq_attention_batched(q, k, v, bias, mask.float()[None], far, 1e6, bias_div=3, split=False)
        got = ops.cross_attention(*(t.unflatten(-1, (heads, d)) for t in (q, k, v)), mask=mask, bias=bias)
        assert (got.flatten(2) - own).abs().max().item() <= 2.0 ** -13 * v.abs().max().item()
