"""Cross attention in bf16 where a batch element is large: the kernels that round
weights to 8 bits, which smaller calls do not reach, against 64 bits; and that an element's
neighbours in the batch do not decide which kernels it gets.

Tolerances: half a step of a result, 2^-14 of the sum of its terms' magnitudes for what is computed in
fp32, 2^-8 of it for the weights' rounding, and in the gradients 2^-8 once more (twice the sizes): P is divided by the
forward pass's sum of rounded weights, off by up to 2^-8 where one weight dominates a row, then P or dS
is rounded itself.  fp32 sums: a lane adds two weights at a time, so a row of N keys makes a chain of at most N / 4
additions (all of them in one split), under 500 u = 2^-15 here; the matrix products add sixteen terms at a time."""

import pytest
import torch
from test_gpu_cross_attention import check, formula, inputs, randn

from boltz_lumi_amd import _native as N
from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu


def eight_bits(case):
    """The rule by which weights have 8 bits: rows of one key head, keys, and an element's products."""
    _, m, n, h, hk, d = case[:6]
    return m * h // hk > 32 and n > 256 and h * m * n * d > 1 << 28


def run(case, gpu, scale):
    q, k, v, mask, bias, g = inputs(case, gpu)
    leaves = [t.requires_grad_() for t in (q, k, v, bias) if t is not None]
    out = ops.cross_attention(q, k, v, mask, bias, scale)
    dout = randn(g, *out.shape, dtype=out.dtype)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        want = formula(q, k, v, mask, bias, scale, dout)
    return zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(), *grads), want)


@pytest.mark.parametrize("case", [  # batch, m, n, heads, kv_heads, dim, mask, bias (per batch element, per head)
    (6, 200, 500, 16, 16, 64, None, None),
    (8, 120, 300, 8, 2, 128, "empty", (0, 1)),
    (8, 150, 513, 16, 16, 48, "some", (1, 1)),
])
def test_a_batch_of_small_elements_rounds_the_result_alone(gpu, case):
    print(f"batch of small elements {case}", flush=True)
    b, m, n, h, _, d = case[:6]
    assert not eight_bits(case) and b * h * m * n * d > 1 << 28
    for name, got, (ref, size) in run((*case, torch.bfloat16), gpu, 2 * case[5] ** -0.5):
        check(got, ref, size, name, weights=False)


LARGE = [  # batch, m, n, heads, kv_heads, dim, mask, bias (per batch element, per head), whether the keys are split
    (1, 910, 1031, 12, 3, 24, None, None, True),
    (4, 700, 1031, 16, 16, 24, "empty", (1, 1), False),
    (1, 700, 801, 10, 10, 48, "some", (1, 1), True),
    (2, 520, 1031, 8, 2, 64, "empty", (0, 1), True),
    (2, 520, 1031, 8, 8, 64, None, (1, 0), True),
    (1, 3000, 1401, 1, 1, 64, "some", None, True),
    (1, 400, 1777, 4, 4, 96, "tail", (0, 0), True),
    (2, 700, 1031, 4, 2, 96, "empty", None, True),
    (2, 300, 901, 8, 4, 128, None, None, True),
    (2, 270, 1000, 8, 1, 128, "empty", (0, 1), True),
    (2, 300, 901, 8, 8, 128, "some", (1, 1), True),
    (1, 65, 5400, 6, 2, 128, "some", None, True),
]


@pytest.mark.parametrize("case", LARGE)
def test_large_elements(gpu, case):
    print(f"large element {case}", flush=True)
    b, m, n, h, hk, d = case[:6]
    assert eight_bits(case)
    assert (N.lib().bmx_cross_attention_workspace_bytes(N.BF16, b, m, n, h, hk, d) > 0) == case[8]
    for name, got, (ref, size) in run((*case[:8], torch.bfloat16), gpu, 0.9 * d ** -0.5):
        check(got, ref, size if name == "out" else size * 2, name)
