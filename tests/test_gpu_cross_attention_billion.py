"""Cross attention over more than 2^30 keys (17 GB each of keys and values): positions and ends of the splits in 32
bits.  All keys but a few of the last ones have logits that leave them no weight, and the few are compared with
64 bits, forward and the queries' gradient; without a mask and with one, many rows and few."""

import pytest
import torch
from test_gpu_cross_attention import check, formula, randn

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu


def test_a_billion_keys(gpu):
    n, tail, d = (1 << 30) + (1 << 23) + 4099, 77, 8  # the last splits start past 2^31 - n
    g = torch.Generator(device=gpu).manual_seed(0)
    k = torch.zeros(1, n, 1, d, device=gpu, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    k[..., 0], v[..., 1] = -64.0, 3.0  # logits of -512 against the tail's few units: weights of zero
    k[:, -tail:], v[:, -tail:] = (randn(g, 1, tail, 1, d, dtype=k.dtype) for _ in range(2))
    mask = torch.zeros(1, n, device=gpu, dtype=torch.bool)
    mask[:, 1 << 29] = True  # of the keys without weight, one to attend
    mask[:, -tail:] = True
    for m in (40, 3):
        q, dout = (randn(g, 1, m, 1, d, dtype=k.dtype) for _ in range(2))
        q[..., 0] = 8.0
        q.requires_grad_()
        for present in (None, mask):
            print(f"{n} keys, {m} queries, mask {present is not None}", flush=True)
            out = ops.cross_attention(q, k, v, present, scale=1.0)
            dq, = torch.autograd.grad(out, q, dout)
            with torch.no_grad():
                want = formula(q, k[:, -tail:], v[:, -tail:], None, None, 1.0, dout)
            check(out.detach(), *want[0], "out")
            check(dq, *want[1], "dq")
