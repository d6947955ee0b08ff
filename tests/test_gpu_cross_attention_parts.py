"""Any part of cross attention's gradients, with sums split or whole and every form of bias, against 64 bits (tolerances:
test_gpu_cross_attention; large elements twice the sizes, test_gpu_cross_attention_large); and calls of two threads at
once, each on a stream of its own.  A bias without a gradient has kernels of its own, which may fuse a product that the
others round (2^-24 of a term); the other choices leave every bit as it is."""

import itertools
import threading

import pytest
import torch
from test_gpu_cross_attention import check, formula, inputs, randn
from test_gpu_cross_attention_large import eight_bits

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", [  # batch, m, n, heads, kv_heads, dim, mask, bias (per batch element, per head), type
    (1, 300, 700, 4, 2, 64, "some", None, torch.bfloat16),
    (2, 300, 700, 4, 2, 48, "some", (0, 1), torch.bfloat16),
    (2, 130, 900, 2, 2, 128, None, (1, 1), torch.bfloat16),
    (2, 7, 500, 2, 1, 32, "empty", (1, 0), torch.float32),
    (2, 520, 1031, 8, 8, 64, None, (1, 1), torch.bfloat16),
])
def test_any_part_of_the_gradients(gpu, case):
    q, k, v, mask, bias, g = inputs(case, gpu)
    tensors = [t for t in (q, k, v, bias) if t is not None]
    dout = randn(g, *q.shape, dtype=q.dtype)

    def grads(wanted):
        leaves = [t.detach().requires_grad_(w) for t, w in zip(tensors, wanted)]
        out = ops.cross_attention(*leaves[:3], mask, leaves[3] if bias is not None else None)
        got = iter(torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dout))
        return [next(got) if w else None for w in wanted]

    with torch.no_grad():
        want = formula(q, k, v, mask, bias, case[5] ** -0.5, dout)[1:]
    large = q.dtype == torch.bfloat16 and eight_bits(case)
    for last in (True, False):  # v, or the bias
        whole = grads([True] * (len(tensors) - 1) + [last])
        for name, got, (ref, size) in zip(("dq", "dk", "dv", "dbias"), whole, want):
            if got is not None:
                check(got, ref, size * 2 if large else size, name, weights=large)
        for wanted in itertools.product((True, False), repeat=len(tensors) - 1):
            if any(wanted) or last:
                for w, some, every in zip((*wanted, last), grads((*wanted, last)), whole):
                    assert some is None if not w else torch.equal(some, every), wanted


def test_two_threads(gpu):
    """Forward and backward of different layouts at once; the plans are shared, workspaces and streams are not."""
    cases = [(2, 70, 600, 4, 2, 64, "some", (0, 1), torch.bfloat16), (1, 40, 900, 2, 2, 32, None, (1, 1), torch.float32)]
    made = [inputs(case, gpu) for case in cases]
    table = torch.randn(32, 4, device=gpu)
    pos, inv = torch.arange(600, device=gpu), torch.rand(16, device=gpu)

    def once(x):
        q, k, v, mask, bias, _ = x
        leaves = [t.detach().requires_grad_() for t in (q, k, v, bias, table)]
        tokens = pos[:q.shape[1]]
        a, _ = ops.qk_norm_rope(leaves[0], None, None, None, tokens, None, inv)
        extra = ops.relative_bias(leaves[4], tokens, pos[:32])
        out = ops.cross_attention(a, leaves[1], leaves[2], mask, leaves[3])
        return out.detach(), *torch.autograd.grad(out.float().sum() + extra.sum(), leaves)

    want = [once(x) for x in made]
    torch.cuda.synchronize()
    failures, ended = [], []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = once(made[i])
                stream.synchronize()
                if not all(torch.equal(x, y) for x, y in zip(want[i], got)):
                    failures.append(i)
        ended.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(ended) == [0, 1] and not failures
