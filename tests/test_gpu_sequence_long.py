"""Gradients of the sequence operators at sizes where a block goes round its loop
many times: a wave's rows of a bias plane, a lane group's heads."""

import pytest
import torch
from test_gpu_qk_norm_rope import test_forward_and_gradients as norm_rope_case
from test_gpu_relative_bias import U, buckets_of

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("buckets,exact,top,bidirectional", [(32, 8, 128, True), (66, 32, 32, True), (32, 16, 128, False)])
def test_relative_bias_table_gradient(gpu, dtype, buckets, exact, top, bidirectional):
    """A wave adds 64 rows of up to 8 columns a lane: chains of at most 512 terms in a bin, then a few dozen over lanes and
    blocks, so within 600 u of the sum of their magnitudes."""
    print(f"table gradient {buckets} {exact} {top} {bidirectional} {dtype}", flush=True)
    heads, m, n = 16, 2048, 2051
    g = torch.Generator(device=gpu).manual_seed(buckets)

    def positions(length):  # steps of one with jumps now and then
        jump = torch.rand(length, generator=g, device=gpu) < 0.01
        return torch.where(jump, torch.randint(-300, 300, (length,), generator=g, device=gpu), 1).cumsum(0)

    q_pos, k_pos = positions(m), positions(n)
    table = torch.randn(buckets, heads, generator=g, device=gpu).to(dtype).requires_grad_()
    bias = ops.relative_bias(table, q_pos, k_pos, exact=exact, max_distance=top, bidirectional=bidirectional)
    index = buckets_of(q_pos, k_pos, buckets, exact, top, bidirectional)
    assert torch.equal(bias.detach(), table.detach()[index].movedim(-1, 0))
    dbias = torch.randn(bias.shape, generator=g, device=gpu).to(dtype)
    dtable, = torch.autograd.grad(bias, table, dbias)
    flat, sums, size = dbias.double().flatten(1), [], []
    for c in range(buckets):
        picked = torch.where(index.flatten() == c, flat, 0.0)
        sums.append(picked.sum(1))
        size.append(picked.abs().sum(1))
    sums, size = torch.stack(sums), torch.stack(size)
    err = (dtable.double() - sums).abs() - 600 * U * size - torch.finfo(dtype).eps / 2 * sums.abs()
    assert bool((err <= 1e-30).all()), err.max().item()


@pytest.mark.parametrize("case", [  # more than 1024 blocks' worth of items in a tensor
    (2, 4099, 777, 32, 8, 128, 64, False, torch.bfloat16, 0),
    (2, 4099, 577, 16, 4, 48, 16, True, torch.float32, 11),
])
def test_norm_rope_gradients(gpu, case):
    norm_rope_case(gpu, case)
