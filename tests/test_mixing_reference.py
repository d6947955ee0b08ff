"""The oracle of the sequence mixing operators: its written-out gradients against automatic ones and against
differences, in fp64 on the CPU."""

import pytest
import torch

from oracle import mixing

F64 = torch.float64


def randn(*shape):
    return torch.randn(*shape, dtype=F64)


def norm_case(gate_tokens):
    x, y, weights = randn(2, 5, 8), randn(2, 5, 8), [randn(8) for _ in range(3)]
    inputs = [x, y, randn(2, gate_tokens, 8), *weights]
    return inputs, lambda *v: mixing.residual_norm(*v, 1e-6), lambda v, back: mixing.residual_norm(*v, 1e-6, *back)


def conv_case(silu):
    inputs = [randn(3, 6, 8), randn(8, 3), randn(8), randn(3, 2, 8)]
    return (inputs, lambda *v: mixing.causal_conv(*v, [6, 1, 0], silu),
            lambda v, back: mixing.causal_conv(*v, [6, 1, 0], silu, *back))


def scan_case(softplus):
    u, dt, z = (randn(3, 5, 16) for _ in range(3))
    if not softplus:
        dt = dt.abs() * 0.3
    inputs = [u, dt, -torch.rand(16, 4, dtype=F64), randn(3, 5, 2, 4), randn(3, 5, 2, 4), randn(16), z,
              randn(16).abs() * 0.1, randn(3, 16, 4)]
    return (inputs, lambda *v: mixing.selective_scan(*v, [5, 2, 0], softplus),
            lambda v, back: mixing.selective_scan(*v, [5, 2, 0], softplus, *back))


CASES = [lambda: norm_case(5), lambda: norm_case(1), lambda: conv_case(True), lambda: conv_case(False),
         lambda: scan_case(True), lambda: scan_case(False)]


@pytest.mark.parametrize("make", CASES)
def test_gradients_against_differences(make):
    """The derivative along a random direction; the error of a central difference of step 1e-5 is about 1e-10 of the
    third derivatives plus 1e-11 of rounding."""
    torch.manual_seed(0)
    inputs, forward, full = make()
    with torch.no_grad():
        results, sizes = full(inputs, [randn(*r.shape) for r in forward(*inputs)[0]])
        torch.manual_seed(1)
        back = [randn(*r.shape) for r in forward(*inputs)[0]]
        results, sizes = full(inputs, back)
        grads = results[len(back):]
        for i, (value, grad) in enumerate(zip(inputs, grads)):
            step = randn(*value.shape)

            def at(h):
                moved = [v + h * step if j == i else v for j, v in enumerate(inputs)]
                return sum((r * g).sum() for r, g in zip(forward(*moved)[0], back))

            want = (at(1e-5) - at(-1e-5)) / 2e-5
            assert abs((grad * step).sum() - want) <= 1e-7 * (1 + abs(want)), i
        for r, s in zip(results, sizes):
            assert (r.abs() <= s * (1 + 1e-12) + 1e-300).all()


@pytest.mark.parametrize("softplus", [True, False])
def test_scan_against_automatic_gradients(softplus):
    torch.manual_seed(2)
    inputs, _, full = scan_case(softplus)
    leaves = [v.requires_grad_() for v in inputs]
    u, dt, A, B, C, D, z, dt_bias, state = leaves
    outs, lasts = [], []
    for i, end in enumerate([5, 2, 0]):
        h, ys = state[i], []
        for t in range(5):
            d = dt[i, t] + dt_bias
            d = torch.log1p(torch.exp(d)) if softplus else d
            if t < end:
                h = torch.exp(d[:, None] * A) * h + (d * u[i, t])[:, None] * B[i, t].repeat_interleave(8, 0)
            y = (h * C[i, t].repeat_interleave(8, 0)).sum(-1) + D * u[i, t]
            ys.append(y * z[i, t] * torch.sigmoid(z[i, t]) * (t < end))
        outs.append(torch.stack(ys))
        lasts.append(h)
    made = [torch.stack(outs), torch.stack(lasts)]
    back = [randn(*r.shape) for r in made]
    want = torch.autograd.grad(made, leaves, back)
    with torch.no_grad():
        results, _ = full(inputs, back)
    for got, expected in zip(results, [*made, *want]):
        assert torch.allclose(got, expected, rtol=1e-11, atol=1e-12)
