"""The gate's gradient of ops.residual_norm where a gate is nearly open: its slope s (1 - s) is about exp(-logit) there,
which one less an s that is already rounded does not hold.

Tolerances: half a step of the result's type, and roundings of 2^-24 relative to the magnitudes that the gradient is made
of, 1 - s among them.  Of s and 1 - s one is about exp(-|logit|), whose exponent is rounded twice (log2(e) and its product):
2 |logit| roundings; everything else (the norms, the gradient of r, the other factor) is under 64, as for the other
gradients, and a sum over rows adds one a row."""

import pytest
import torch

from boltz_lumi_amd import ops
from oracle import mixing
from mixing_cases import BF16, FP32, assert_close, fp64, leaf, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 264, 1024, 2048, 4104])
@pytest.mark.parametrize("stream,dtype", [(FP32, FP32), (FP32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("kind", ["token", "sample"])
@pytest.mark.parametrize("post,pre", [(True, True), (False, False)])
def test_nearly_open_and_shut(gpu, d, stream, dtype, kind, post, pre):
    g = torch.Generator().manual_seed(d)
    b, t, most, eps = 2, 13, 60.0, 1e-6
    x, y = randn(g, b, t, d, dtype=stream, scale=2.0), randn(g, b, t, d, dtype=dtype)
    gate = torch.linspace(-most, most, b * d).view(b, 1, d)
    gate = (gate if kind == "sample" else gate.repeat(1, t, 1)).to(dtype)
    yw, k, w = (randn(g, d, scale=0.3, shift=1.0) for _ in range(3))
    inputs = [x, y, gate, yw if post else None, k, w if pre else None]
    back = [randn(g, b, t, d, dtype=stream), randn(g, b, t, d, dtype=dtype)]
    leaves = [leaf(v, gpu) for v in inputs]
    made = ops.residual_norm(*leaves, eps=eps, post_norm=post, pre_norm=pre)
    made = made if pre else (made,)
    got, = torch.autograd.grad(made, leaves[2], [v.to(gpu) for v in back[:len(made)]])
    with torch.no_grad():
        results, sizes = mixing.residual_norm(*map(fp64, inputs), eps, *map(fp64, back), post_norm=post, pre_norm=pre)
    y, gate = fp64(y), fp64(gate)
    n = y * (y.square().mean(-1, keepdim=True) + eps).rsqrt() * fp64(yw) if post else y
    dR, away = results[1 + pre], torch.sigmoid(-gate)  # 1 - s, which fp64 does not hold past 36 either
    want = dR * fp64(k) * torch.sigmoid(gate) * n * away
    want = want.sum(1, keepdim=True) if kind == "sample" else want
    assert_close("dgate", got, want, sizes[3 + pre] * away, 64 + 2 * most + t)
