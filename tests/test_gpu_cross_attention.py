"""Cross attention (ops.cross_attention) against its formula in 64 bits: values,
gradients, masks that leave rows empty, shared heads and biases, layouts.

Tolerances.  u = 2^-24.  fp32: a logit is a sum of D products (D u of |q| . |k|, times scale), a weight's
relative error is that of its logits plus the exponential's 2 u and the change of base (u of the logits'
range), sums over N keys add at most N / 8 in a chain: with these inputs under 2^-14 of the sum of magnitudes.
bf16: weights (and their gradients) are rounded once before the product over them, half a
step (2^-8) of each, and the result once more; the output and dV, dQ, dK are compared with 2^-8 of the sum
of the magnitudes of their terms plus 2^-8 of themselves, on top of the fp32 part. Up to 256 keys, and in small calls,
weights have 16 bits: what that leaves, 2^-16 of each, is inside the fp32 part's 2^-14 (whose own share with
D = 128 and logits of a few units stays below 2^-15)."""

import math

import pytest
import torch

from boltz_lumi_amd import _native as N
from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def formula(q, k, v, mask, bias, scale, dout=None):
    """out, and with dout (dq, dk, dv, dbias), in fp64; beside each the sum of the magnitudes of its terms."""
    b, m, h, d = q.shape
    hk = k.shape[2]
    g = h // hk
    q, k, v = (t.double().transpose(1, 2) for t in (q, k, v))
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    if bias is not None:
        s = s + bias.double()
    if mask is not None:
        keep = mask.expand(b, -1)[:, None, None]
        s = s.masked_fill(~keep, -math.inf)
        k, v = (t.masked_fill(~keep.transpose(2, 3), 0.0) for t in (k, v))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out = torch.matmul(p, v)
    size = torch.matmul(p, v.abs())
    back = [(t.transpose(1, 2)) for t in (out, size)]
    if dout is None:
        return back
    do = dout.double().transpose(1, 2)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (do * out).sum(-1, keepdim=True))
    # what a relative error of every weight and of every rounded ds can move ds by
    ds_size = p * (dp.abs() + torch.matmul(p, dp.abs().transpose(2, 3)).diagonal(dim1=2, dim2=3)[..., None])

    def heads(t):  # sum over the group, back to [B, T, Hk, D]
        return t.unflatten(1, (hk, g)).sum(2).transpose(1, 2)

    dq = [torch.matmul(x, y).transpose(1, 2) * scale for x, y in ((ds, k), (ds_size, k.abs()))]
    dk = [heads(torch.matmul(x.transpose(2, 3), y) * scale) for x, y in ((ds, q), (ds_size, q.abs()))]
    dv = [heads(torch.matmul(p.transpose(2, 3), y)) for y in (do, do.abs())]
    if bias is None:
        return back, dq, dk, dv
    axes = [i for i in (0, 1) if bias.shape[i] == 1]
    dbias = [x.sum(axes, keepdim=True) if axes else x for x in (ds, ds_size)]
    return back, dq, dk, dv, dbias


def check(got, want, size, what, weights=True):
    """weights: bf16 weights are rounded to its 8 bits."""
    assert got.shape == want.shape, what
    step = half_step(got.dtype)
    near = 2.0 ** -14 + (step if weights and got.dtype == torch.bfloat16 else 0)
    err = (got.double() - want).abs() - near * size - step * want.abs()
    assert bool((err <= 1e-30).all()), f"{what}: {err.max().item()} past the bound"


def randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=g.device).to(dtype)


def inputs(case, gpu, seed=0):
    b, m, n, h, hk, d, masked, bias, dtype = case
    g = torch.Generator(device=gpu).manual_seed(seed + m + n)
    q, k, v = (randn(g, b, t, x, d, dtype=dtype) for t, x in ((m, h), (n, hk), (n, hk)))
    mask = None
    if masked:
        mask = torch.rand(b, n, generator=g, device=gpu) < 0.6
        if masked == "tail":
            mask = torch.arange(n, device=gpu) < torch.randint(0, n + 1, (b, 1), generator=g, device=gpu)
        if masked == "empty":
            mask[-1] = False
    if bias is not None:
        bias = randn(g, *(s if w else 1 for s, w in zip((b, h), bias)), m, n, dtype=dtype)
    return q, k, v, mask, bias, g


CASES = [  # batch, m, n, heads, kv_heads, dim, mask, bias (per batch element, per head), type
    (1, 1, 1, 1, 1, 8, None, None, torch.bfloat16),
    (1, 1, 1, 2, 1, 16, None, (1, 1), torch.float32),
    (2, 1, 117, 16, 16, 24, "some", None, torch.float32),
    (3, 1, 700, 8, 2, 128, "tail", (0, 1), torch.bfloat16),
    (2, 5, 4200, 12, 2, 64, "empty", None, torch.bfloat16),
    (1, 33, 31, 3, 3, 48, "some", (1, 0), torch.bfloat16),
    (2, 130, 65, 4, 2, 32, "empty", (0, 0), torch.float32),
    (2, 129, 257, 4, 1, 96, "tail", (0, 1), torch.bfloat16),
    (1, 300, 190, 2, 2, 128, None, (1, 1), torch.bfloat16),
    (1, 70, 300, 4, 2, 128, "some", (0, 1), torch.float32),
    (2, 65, 130, 2, 2, 96, None, None, torch.float32),
    (1, 257, 513, 6, 2, 64, None, None, torch.bfloat16),
    (5, 64, 64, 2, 2, 40, "some", (0, 1), torch.bfloat16),
    (1, 17, 8300, 1, 1, 64, "some", None, torch.bfloat16),
    (1, 200, 4161, 2, 1, 64, "tail", None, torch.float32),
    (2, 140, 300, 4, 2, 128, "empty", (1, 0), torch.bfloat16),
]


@pytest.mark.parametrize("case", CASES)
def test_values_and_gradients(gpu, case):
    print(f"cross_attention {case}", flush=True)
    q, k, v, mask, bias, g = inputs(case, gpu)
    scale = 0.9 * case[5] ** -0.5
    with torch.no_grad():
        got = ops.cross_attention(q, k, v, mask, bias, scale)
    leaves = [t.requires_grad_() for t in (q, k, v, bias) if t is not None]
    out = ops.cross_attention(q, k, v, mask, bias, scale)
    assert out.is_contiguous() and torch.equal(out.detach(), got)
    dout = randn(g, *out.shape, dtype=out.dtype)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        want = formula(q, k, v, mask, bias, scale, dout)
    check(got, *want[0], "out")
    for name, have, (ref, size) in zip(("dq", "dk", "dv", "dbias"), grads, want[1:]):
        check(have, ref, size, name)


def test_one_key_has_no_logit_gradient(gpu):
    """The weight of a single key is 1 whatever its logit: out is v itself, dq and dk vanish to fp32 rounding."""
    g = torch.Generator(device=gpu).manual_seed(5)
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v = (randn(g, 2, t, 4, 64, dtype=dtype).requires_grad_() for t in (40, 1, 1))
        out = ops.cross_attention(q, k, v)
        assert torch.equal(out.detach(), v.detach().expand_as(out))
        dout = randn(g, *out.shape, dtype=dtype)
        dq, dk, _ = torch.autograd.grad(out, (q, k, v), dout)
        # dP - delta: two sums of 64 products of dO and v in another order
        size = (dout.double().abs() * v.detach().double().abs()).sum(-1, keepdim=True) * 64 * U
        assert bool((dq.double().abs() <= size * k.detach().double().abs() + 1e-30).all())
        assert bool((dk.double().abs() <= (size * q.detach().double().abs()).sum(1, keepdim=True) + 1e-30).all())


@pytest.mark.parametrize("case", [  # few keys; then small calls over many
    (2, 300, 2, 4, 2, 48, None, (0, 1), torch.bfloat16),
    (5, 30, 23, 2, 2, 32, "some", (1, 1), torch.bfloat16),
    (1, 200, 256, 2, 1, 128, "tail", None, torch.bfloat16),
    (2, 1, 97, 4, 1, 96, None, None, torch.bfloat16),
    (1, 40, 900, 2, 2, 64, "some", None, torch.bfloat16),
    (1, 5, 2500, 2, 1, 24, None, (1, 0), torch.bfloat16),
])
def test_small_calls_round_the_result_alone(gpu, case):
    q, k, v, mask, bias, g = inputs(case, gpu)
    scale = case[5] ** -0.5
    leaves = [t.requires_grad_() for t in (q, k, v, bias) if t is not None]
    out = ops.cross_attention(q, k, v, mask, bias, scale)
    dout = randn(g, *out.shape, dtype=out.dtype)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        want = formula(q, k, v, mask, bias, scale, dout)
    for name, have, (ref, size) in zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(), *grads), want):
        check(have, ref, size, name, weights=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 60, 150])
def test_masks_hide_anything(gpu, dtype, m):
    """NaN, infinities and the lowest value in left-out keys change nothing, in values or gradients; rows whose
    keys are all left out (by the mask or by -inf) give zeros; rows biased by the lowest value throughout attend
    evenly, as adding that value to their logits does."""
    b, n, h, d = 3, 150, 2, 32
    g = torch.Generator(device=gpu).manual_seed(6)
    q, k, v = (randn(g, b, t, h, d, dtype=dtype) for t in (m, n, n))
    mask = torch.rand(b, n, generator=g, device=gpu) < 0.5
    mask[1] = False
    low = torch.finfo(dtype).min
    bias = randn(g, 1, h, m, n, dtype=dtype)
    bias[0, 0, 0] = low
    bias[0, 1, m - 1] = -math.inf
    bias[0, 0, m // 2, ::3] = low if m > 1 else 0
    dout = randn(g, b, m, h, d, dtype=dtype)

    def run(k, v, bias):
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, bias)]
        out = ops.cross_attention(*leaves[:3], mask, leaves[3])
        return out.detach(), *torch.autograd.grad(out, leaves, dout)

    clean = run(k, v, bias)
    off = ~mask[:, :, None, None]
    dirty = run(torch.where(off, math.nan, k), torch.where(off, math.inf, v), bias)
    for a, c in zip(clean, dirty):
        assert torch.isfinite(a).all() and torch.equal(a, c)
    out, dq, dk, dv, dbias = clean
    assert not out[1].any() and not dq[1].any() and not dk[1].any() and not dv[1].any()
    assert not out[:, m - 1, 1].any() and not dbias[0, 1, m - 1].any()
    assert not dk.masked_select(off).any() and not dv.masked_select(off).any()
    # Query 0 of head 0: the lowest value at every key (m = 1: 0 at every third key, which then share the weight).
    # Against it q k^T is below half a step, so the keys at its maximum weigh the same for m > 1; for m = 1 their
    # own logits remain.
    for i in (0, 2):
        keys = mask[i] & (bias[0, 0, 0] == bias[0, 0, 0].max())
        x = v[i][keys][:, 0].double()
        if m > 1:
            weights = torch.full_like(x[:, 0], 1 / x.shape[0])
        else:
            weights = torch.softmax(k[i][keys][:, 0].double() @ q[i, 0, 0].double() / math.sqrt(d), 0)
        check(out[i, 0, 0], weights @ x, weights @ x.abs(), "lowest")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 40), (1, 3000), (50, 40), (200, 700)])
def test_nan_is_kept(gpu, dtype, m, n):
    """NaN in a query or in a present key shows in every result it belongs to, and in no other row."""
    g = torch.Generator(device=gpu).manual_seed(9)
    q, k, v = (randn(g, 2, t, 2, 32, dtype=dtype) for t in (m, n, n))
    dout = torch.ones_like(q)
    q[0, m - 1, 1, 3] = math.nan
    k[1, n // 2, 0, 5] = math.nan
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    want = torch.zeros(2, m, 2, dtype=torch.bool, device=gpu)
    want[0, m - 1, 1] = True
    want[1, :, 0] = True
    for t in (out, dq):
        bad = torch.isnan(t)
        assert torch.equal(bad.all(-1), want) and torch.equal(bad.any(-1), want)
    heads = torch.tensor([[False, True], [True, False]], device=gpu)[:, None].expand(2, n, 2)
    for t in (dk, dv):
        assert torch.equal(torch.isnan(t).any(-1), heads)


def test_layouts(gpu):
    """Column slices of joint projections, head-major tensors, odd storage offsets, a bias and a mask by strides: the
    same bits as dense operands."""
    b, m, n, h, hk, d = 2, 37, 53, 4, 2, 24
    g = torch.Generator(device=gpu).manual_seed(7)
    kv = randn(g, b, n, 2 * hk * d, dtype=torch.bfloat16)
    q = randn(g, b, h, m, d, dtype=torch.bfloat16).transpose(1, 2)
    k, v = (kv[..., i * hk * d:(i + 1) * hk * d].unflatten(-1, (hk, d)) for i in (0, 1))
    wide = torch.rand(b, 2 * n + 3, generator=g, device=gpu) < 0.7
    mask = wide[:, 3:3 + 2 * n:2]
    bias = randn(g, h, m, n + 5, dtype=torch.bfloat16)[None, ..., 3:3 + n]
    with torch.no_grad():
        dense = ops.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), mask.contiguous(), bias.contiguous())
        assert torch.equal(ops.cross_attention(q, k, v, mask, bias), dense)
        odd = torch.empty(q.numel() + 1, device=gpu, dtype=q.dtype)[1:].view(b, m, h, d).copy_(q)
        assert torch.equal(ops.cross_attention(odd, k, v, mask, bias), dense)
        tall = v.transpose(1, 3).contiguous().transpose(1, 3)  # strided channels
        assert torch.equal(ops.cross_attention(q, k, tall, mask, bias), dense)
        one = ops.cross_attention(q, k, v, mask[:1], None)
        assert torch.equal(one, ops.cross_attention(q, k, v, mask[0], None))
        assert torch.equal(one, ops.cross_attention(q, k, v, mask[:1].expand(b, n), None))
    leaves = [t.detach().requires_grad_() for t in (q, k, v, bias)]
    out = ops.cross_attention(*leaves[:3], mask, leaves[3])
    some = torch.autograd.grad(out.sum(), leaves[1:3])  # an expanded gradient, a part of the leaves
    full = torch.autograd.grad(ops.cross_attention(*leaves[:3], mask, leaves[3]), leaves, torch.ones_like(out))
    assert all(torch.equal(x, y) for x, y in zip(some, full[1:3]))


def test_empty_sizes(gpu):
    for b, m, n in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = (torch.randn(b, t, 2, 16, device=gpu, requires_grad=True) for t in (m, n, n))
        bias = torch.randn(1, 2, m, n, device=gpu, requires_grad=True)
        out = ops.cross_attention(q, k, v, None, bias)
        assert out.shape == q.shape and not out.any()
        for t, gt in zip((q, k, v, bias), torch.autograd.grad(out, (q, k, v, bias), torch.ones_like(out))):
            assert gt.shape == t.shape and not gt.any()


def test_differences(gpu):
    """Central differences of the fp32 forward along each gradient (h = 2^-5) to 1%."""
    q, k, v, mask, bias, g = inputs((2, 9, 21, 4, 2, 16, "some", (0, 1), torch.float32), gpu)
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    out = ops.cross_attention(q, k, v, mask, bias)
    dout = randn(g, *out.shape, dtype=out.dtype)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        for i, dx in enumerate(grads):
            step, ends = dx / dx.abs().max() / 32, []
            for sign in (1, -1):
                x = [t + sign * step if j == i else t for j, t in enumerate(leaves)]
                ends.append((ops.cross_attention(*x[:3], mask, x[3]).double() * dout).sum())
            slope, want = (ends[0] - ends[1]).item() / 2, (dx.double() * step).sum().item()
            assert abs(slope - want) <= 1e-2 * abs(want), (i, slope, want)


def test_same_bits_streams_and_graph(gpu):
    """The same bits on every run, on another stream, and from a captured forward and backward replayed with eager
    work between."""
    q, k, v, mask, bias, g = inputs((2, 70, 600, 4, 2, 64, "some", (0, 1), torch.bfloat16), gpu)
    dout = randn(g, *q.shape, dtype=q.dtype)

    def once():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, bias)]
        out = ops.cross_attention(*leaves[:3], mask, leaves[3])
        return out.detach(), *torch.autograd.grad(out, leaves, dout)

    def token():
        with torch.no_grad():
            return ops.cross_attention(q[:, :1], k, v, mask, None)

    want, single = once(), token()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(x, y) for x, y in zip(want, once()))
        token()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, one = once(), token()
    for shift in (0.0, 0.5, -1.0):
        q.copy_(q + shift)
        want, single = once(), token()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, held)) and torch.equal(single, one)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 32)])
@pytest.mark.parametrize("axes", [(0,), (1,), (0, 1)])
def test_native_dbias_shared_by_own_biases(gpu, dtype, dim, axes):
    """The C entry sums dbias over axes along which the bias itself differs."""
    b, m, n, h, hk = 3, 70, 150, 4, 2
    q, k, v, mask, bias, g = inputs((b, m, n, h, hk, dim, "tail", (1, 1), dtype), gpu)
    mask[1] = False
    scale, dout = dim ** -0.5, randn(g, b, m, h, dim, dtype=dtype)
    lo, out, stats = torch.empty_like(q), torch.empty_like(q), torch.empty(b, h, m, 2, device=gpu)
    dbias = torch.full([1 if i in axes else s for i, s in enumerate((b, h))] + [m, n], math.nan, device=gpu, dtype=dtype)
    code = N.F32 if dtype == torch.float32 else N.BF16
    shape = N.int64_array([b, m, n, h, hk, dim])
    strides = N.int64_array([*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], n, *bias.stride()[:3]])
    steps = N.int64_array([0 if i in axes else st for i, st in enumerate(dbias.stride()[:3])])
    size = max(N.lib().bmx_cross_attention_workspace_bytes(code, b, m, n, h, hk, dim),
               N.lib().bmx_cross_attention_bwd_workspace_bytes(b, m, n, h, hk, dim))
    ws, stream = torch.empty(size, device=gpu, dtype=torch.uint8), torch.cuda.current_stream().cuda_stream
    head = (*(t.data_ptr() for t in (q, k, v, mask, bias)), code, shape, strides, scale, out.data_ptr(), lo.data_ptr(),
            stats.data_ptr())
    N.call("bmx_cross_attention_fwd", *head, ws.data_ptr(), size, stream)
    N.call("bmx_cross_attention_bwd", *head, dout.data_ptr(), None, None, None, dbias.data_ptr(), steps, ws.data_ptr(), size,
           stream)
    ref, sizes = (t.sum(axes, keepdim=True) for t in formula(q, k, v, mask, bias, scale, dout)[4])
    check(dbias, ref, sizes, "dbias", weights=False)


def test_long_cache_offsets(gpu):
    """Keys whose offsets pass 2^31 elements: one query over the last of a long, wide cache."""
    n, hk, d = 1 << 21, 9, 128  # 2.4e9 elements
    k = torch.zeros(1, n, hk, d, device=gpu, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    g = torch.Generator(device=gpu).manual_seed(8)
    tail = 70
    k[:, -tail:], v[:, -tail:] = (randn(g, 1, tail, hk, d, dtype=k.dtype) for _ in range(2))
    mask = torch.zeros(1, n, device=gpu, dtype=torch.bool)
    mask[:, -tail:] = True
    q = randn(g, 1, 1, hk, d, dtype=k.dtype)
    with torch.no_grad():
        got = ops.cross_attention(q, k, v, mask)
        assert torch.equal(got[:, :, -1:], ops.cross_attention(q[:, :, -1:], k[:, :, -1:], v[:, :, -1:], mask))
        check(got, *formula(q, k[:, -tail:], v[:, -tail:], None, None, d ** -0.5), "long")


def test_refusals(gpu):
    q, k, v, mask, bias, _ = inputs((2, 5, 7, 4, 2, 32, "some", (0, 1), torch.float32), gpu)
    good = dict(q=q, k=k, v=v, mask=mask, bias=bias)
    for change, text in [
        ({"q": q[0]}, "shape"), ({"q": q.half()}, "dtype"), ({"k": k.bfloat16()}, "match q"), ({"v": v[:, :6]}, "match q"),
        ({"k": k[:1], "v": v[:1]}, "match q"), ({"k": k[..., :24], "v": v[..., :24]}, "match q"),
        ({"q": q[..., :20], "k": k[..., :20], "v": v[..., :20]}, "multiple of 8"),
        ({"q": q[:, :, :3]}, "multiple of the key heads"), ({"mask": mask.float()}, "bool mask"),
        ({"mask": mask[:, :6]}, "bool mask"), ({"bias": bias.bfloat16()}, "bias"), ({"bias": bias[..., :1]}, "bias"),
        ({"bias": bias[0]}, "bias"), ({"bias": bias[:, :3]}, "bias"), ({"scale": 0.0}, "scale"),
        ({"scale": float("inf")}, "scale"), ({"scale": float("nan")}, "scale"), ({"k": k.cpu()}, "CUDA"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            ops.cross_attention(**{**good, **change})
    wide = torch.zeros(1, 2, 1, 136, device=gpu)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.cross_attention(wide, wide, wide)
