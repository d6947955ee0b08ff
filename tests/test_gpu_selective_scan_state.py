"""The first state of ops.selective_scan under autograd: its gradient does not read it, so it may move on in place between
the forward and the backward pass (a decoder's state that a training step starts from)."""

import pytest
import torch

from boltz_lumi_amd import ops
from mixing_cases import BF16, FP32, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1, 70])
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("learned", [False, True])
def test_state_moves_on_before_backward(gpu, t, dtype, learned):
    g = torch.Generator().manual_seed(t)
    b, c, n = 2, 24, 16
    u, dt = (randn(g, b, t, c, dtype=dtype).to(gpu) for _ in range(2))
    B, C = (randn(g, b, t, 1, n, dtype=dtype).to(gpu) for _ in range(2))
    A, state = -randn(g, c, n).abs().to(gpu), randn(g, b, c, n).to(gpu)
    back = [randn(g, b, t, c, dtype=dtype).to(gpu), randn(g, b, c, n).to(gpu)]

    def gradients(move):
        leaves = [v.clone().requires_grad_() for v in (u, dt, A, B, C)]
        first = state.clone().requires_grad_(learned)
        made = ops.selective_scan(*leaves, state=first, return_state=True)
        if move:
            with torch.no_grad():
                ops.selective_scan(*leaves, state=first, state_out=first)
        return torch.autograd.grad(made, leaves + [first] * learned, back)

    for kept, moved in zip(gradients(False), gradients(True)):
        assert torch.equal(kept, moved)


@pytest.mark.parametrize("last", [False, True])
def test_no_tokens(gpu, last):
    """Without tokens the state's gradient is the last one's, or zeros where nothing came from that."""
    rows, maps = torch.zeros(2, 0, 8, device=gpu), torch.zeros(2, 0, 1, 8, device=gpu)
    state = torch.ones(2, 8, 8, device=gpu, requires_grad=True)
    out, after = ops.selective_scan(rows, rows, -torch.ones(8, 8, device=gpu), maps, maps, state=state, return_state=True)
    grad, = torch.autograd.grad(after.sum() * 3 if last else out.sum(), state)
    assert torch.equal(grad, torch.full_like(state, 3.0 if last else 0.0))
