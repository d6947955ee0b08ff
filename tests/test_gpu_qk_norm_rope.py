"""Query / key norm with rotation (ops.qk_norm_rope) against its formula in 64
bits, forward and gradients.

Tolerances, u = 2^-24: the sum of squares has at most 13 additions in a chain (8 values
of a lane, 5 exchanges), the root halves its error, and the products, the angle and
the rotation add a few u each, so a result is within 32 u of the row's largest
normalised value before it is rounded (half a step of its type).  The gradient
chains two such sums: 128 u of its row's scale.  A weight gradient adds at
most 256 terms in a chain here: 256 u of the sum of their magnitudes."""

import pytest
import torch

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, w, pos, inv_freq, eps, interleaved):
    """(result, normalised values) in the dtype of x (fp64)."""
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n = n if w is None else n * w
    if inv_freq is None:
        return n, n
    r = inv_freq.numel()
    angle = (pos.double()[..., None] * inv_freq.double())[..., None, :]  # [(B,) T, 1, R]
    c, s = angle.cos(), angle.sin()
    a, b = (n[..., 0:2 * r:2], n[..., 1:2 * r:2]) if interleaved else (n[..., :r], n[..., r:2 * r])
    a, b = a * c - b * s, a * s + b * c
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, n[..., 2 * r:]], -1), n


def half_step(t):
    return torch.finfo(t.dtype).eps / 2


def check(got, want, bound, what):
    assert got.shape == want.shape
    err = (got.double() - want).abs() - bound - half_step(got) * want.abs()
    assert bool((err <= 1e-30).all()), f"{what}: {err.max().item()} past the bound"


CASES = [  # batch, m, n, heads, kv_heads, dim, rotated pairs, interleaved, dtype, start
    (1, 1, 1, 32, 8, 128, 64, False, torch.bfloat16, 1000003),
    (2, 33, 7, 3, 1, 24, 12, False, torch.float32, 0),
    (1, 5, 0, 2, 4, 8, 4, True, torch.float32, 3),
    (2, 70, 41, 16, 16, 48, 16, True, torch.bfloat16, 0),
    (3, 17, 19, 5, 2, 96, 24, False, torch.bfloat16, 7),
    (1, 300, 301, 6, 3, 256, 128, False, torch.float32, -150),
    (2, 1100, 800, 16, 4, 64, 32, True, torch.float32, 0),
    (1, 64, 64, 7, 7, 16, 0, False, torch.float32, 0),
]


def make(case, gpu, seed=0):
    b, m, n, h, hk, d, r, interleaved, dtype, start = case
    g = torch.Generator(device=gpu).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=gpu)

    q, k = (randn(b, m, h, d) * 2).to(dtype), (randn(b, n, hk, d) * 0.3).to(dtype)
    qw, kw = (1 + 0.2 * randn(d)).to(dtype), (1 + 0.2 * randn(d)).to(dtype)
    q_pos = torch.arange(m, device=gpu) + start
    k_pos = torch.arange(n, device=gpu) + start
    inv = None if r == 0 else 10000.0 ** (-torch.arange(r, device=gpu, dtype=torch.float64) / r)
    return q, k, qw, kw, q_pos, k_pos, inv


@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(gpu, case):
    print(f"qk_norm_rope {case}", flush=True)
    q, k, qw, kw, q_pos, k_pos, inv = make(case, gpu)
    interleaved, eps = case[7], 1e-6
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    out = ops.qk_norm_rope(q, k, qw, kw, q_pos, k_pos, inv, eps=eps, interleaved=interleaved)
    g = torch.Generator(device=gpu).manual_seed(1)
    dout = [torch.randn(o.shape, generator=g, device=gpu).to(o.dtype) for o in out]
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        plain = ops.qk_norm_rope(q, k, qw, kw, q_pos, k_pos, inv, eps=eps, interleaved=interleaved)
    for i, (x, w, pos) in enumerate(((q, qw, q_pos), (k, kw, k_pos))):
        assert torch.equal(plain[i], out[i])
        x64, w64 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        y, n = reference(x64, w64, pos, inv, eps, interleaved)
        top = n.abs().amax(-1, keepdim=True)
        check(out[i].detach(), y.detach(), 32 * U * top, "result")
        dx, dw = torch.autograd.grad(y, (x64, w64), dout[i].double())
        root = (x64.square().mean(-1, keepdim=True) + eps).rsqrt()
        scale = root * dout[i].double().abs().amax(-1, keepdim=True) * w64.abs().max() * 2
        check(grads[i], dx, 128 * U * scale * (1 + top * top), "dx")
        # g x r: magnitudes through the rotation are at most sqrt(2) of the pair's
        terms = (dout[i].double().abs().amax(-1, keepdim=True) * 1.5 * (n / w64).abs()).sum((0, 1, 2))
        check(grads[2 + i], dw, 256 * U * terms, "dw")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_positions_and_absent_operands(gpu, dtype):
    """Column slices of one projection, per-element int32 positions, fp32 weights, no weights, no rotation, no keys."""
    g = torch.Generator(device=gpu).manual_seed(2)
    b, m, h, hk, d = 2, 37, 4, 2, 32
    proj = torch.randn(b, m, (h + 2 * hk) * d + 6, generator=g, device=gpu).to(dtype)
    q = proj[..., :h * d].unflatten(-1, (h, d))
    k = proj[..., h * d:(h + hk) * d].unflatten(-1, (hk, d))
    pos = torch.randint(-2000, 2000, (b, m), generator=g, device=gpu, dtype=torch.int32)
    inv = torch.rand(8, generator=g, device=gpu)
    w = torch.rand(d, generator=g, device=gpu) + 0.5
    with torch.no_grad():
        got = ops.qk_norm_rope(q, k, w, None, pos, pos[0], inv, eps=1e-5)
        for o, x, wx, px in zip(got, (q, k), (w, None), (pos, pos[0])):
            y, n = reference(x.double(), None if wx is None else wx.double(), px, inv, 1e-5, False)
            check(o, y, 32 * U * n.abs().amax(-1, keepdim=True), "strided")
        alone, none = ops.qk_norm_rope(q, None, w, None, pos, None, inv, eps=1e-5)
        assert none is None and torch.equal(alone, got[0])
        odd = torch.empty(b * m * h * d + 1, device=gpu, dtype=dtype)[1:].view(b, m, h, d).copy_(q)  # unaligned
        assert torch.equal(ops.qk_norm_rope(odd, None, w, None, pos, None, inv, eps=1e-5)[0], got[0])
        flat, _ = ops.qk_norm_rope(q, None, None, None, None, None, None, eps=1e-5)
        n = reference(q.double(), None, None, None, 1e-5, False)[0]
        check(flat, n, 32 * U * n.abs().amax(-1, keepdim=True), "no rotation")


def test_gradient_of_one_result_and_differences(gpu):
    """Only q' used: k and its weight get no gradient.  Central differences (h = 2^-6 along a direction)
    agree to 1%: their truncation is h^2 / 6 of the third derivative, their rounding u / h of the values."""
    q, k, qw, kw, q_pos, k_pos, inv = make((1, 9, 5, 4, 2, 64, 32, False, torch.float32, 11), gpu)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    g = torch.Generator(device=gpu).manual_seed(3)
    out, _ = ops.qk_norm_rope(*leaves, q_pos, k_pos, inv)
    dout = torch.randn(out.shape, generator=g, device=gpu)
    dq, dk, dqw, dkw = torch.autograd.grad(out, leaves, dout, allow_unused=True)
    assert dk is None and dkw is None
    with torch.no_grad():
        for x, dx in ((q, dq), (qw, dqw)):
            v, h = dx / dx.abs().max(), 2.0 ** -6
            ends = []
            for sign in (1, -1):
                args = [q, k, qw, kw]
                args[0 if x is q else 2] = x + sign * h * v
                ends.append((ops.qk_norm_rope(*args, q_pos, k_pos, inv)[0].double() * dout).sum())
            slope, want = ((ends[0] - ends[1]) / (2 * h)).item(), (dx.double() * v).sum().item()
            assert abs(slope - want) <= 1e-2 * abs(want), (slope, want)


def test_same_bits_and_another_stream(gpu):
    q, k, qw, kw, q_pos, k_pos, inv = make((2, 1100, 900, 8, 4, 64, 32, False, torch.bfloat16, 0), gpu)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    dout = [torch.ones_like(q), torch.ones_like(k)]

    def once():
        return torch.autograd.grad(ops.qk_norm_rope(*leaves, q_pos, k_pos, inv), leaves, dout)

    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_refusals(gpu):
    q, k, qw, kw, q_pos, k_pos, inv = make((1, 4, 4, 2, 2, 32, 16, False, torch.float32, 0), gpu)
    good = dict(q=q, k=k, q_weight=qw, k_weight=kw, q_pos=q_pos, k_pos=k_pos, inv_freq=inv)
    for change, text in [
        ({"q": q[0]}, "shape"), ({"q": q.half()}, "dtype"), ({"q": q[..., :20], "k": k[..., :20]}, "multiple of 8"),
        ({"k": k.bfloat16()}, "match q"), ({"k": k[..., :24]}, "match q"), ({"k": None}, "needs k"),
        ({"q_weight": qw[:16]}, "weights"), ({"q_weight": qw.half()}, "weights"),
        ({"q_pos": q_pos.float()}, "int32 or int64"), ({"q_pos": q_pos[:3]}, "shape"), ({"q_pos": None}, "int32"),
        ({"k_pos": k_pos.int()}, "share"), ({"inv_freq": inv[:3]}, "multiple of 4"),
        ({"inv_freq": torch.cat([inv, inv[:4]])}, "multiple of 4"), ({"eps": 0.0}, "eps"), ({"q": q.cpu()}, "CUDA"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            ops.qk_norm_rope(**{**good, **change})
