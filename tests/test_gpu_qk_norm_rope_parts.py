"""Gradients of qk_norm_rope where only some are wanted: the same bits as all of them, and neither memory nor work
for the others; NULL gradients at the C entry."""

import itertools

import pytest
import torch
from test_gpu_qk_norm_rope import make

from boltz_lumi_amd import _native as N
from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu
CASE = (2, 300, 260, 8, 4, 64, 32, False, torch.bfloat16, 5)


def test_any_part_of_the_gradients(gpu):
    q, k, qw, kw, q_pos, k_pos, inv = make(CASE, gpu)
    dout = [torch.randn_like(t) for t in (q, k)]

    def grads(wanted):
        leaves = [t.detach().requires_grad_(w) for t, w in zip((q, k, qw, kw), wanted)]
        out = ops.qk_norm_rope(*leaves, q_pos, k_pos, inv)
        picked = [t for t in leaves if t.requires_grad]
        pairs = [(o, d) for o, d in zip(out, dout) if o.requires_grad]
        got = iter(torch.autograd.grad([o for o, _ in pairs], picked, [d for _, d in pairs]))
        return [next(got) if w else None for w in wanted]

    whole = grads((True,) * 4)
    for wanted in itertools.product((True, False), repeat=4):
        if any(wanted):
            for w, some, every in zip(wanted, grads(wanted), whole):
                assert some is None if not w else torch.equal(some, every), wanted


def test_weights_alone_take_no_memory_for_the_rest(gpu):
    q, k, qw, kw, q_pos, k_pos, inv = make((2, 4096, 4096, 8, 8, 128, 64, False, torch.bfloat16, 0), gpu)
    weights = [t.requires_grad_() for t in (qw, kw)]
    out = ops.qk_norm_rope(q, k, *weights, q_pos, k_pos, inv)
    dout = [torch.ones_like(o) for o in out]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    torch.autograd.grad(out, weights, dout)
    assert torch.cuda.max_memory_allocated() - before < q.numel() * 2  # the workspace is 1 MB, dq alone 17


def test_native_null_gradients(gpu):
    """Every choice of NULL pointers writes the others as the full call does; a tensor with neither gradient may have
    a NULL dy."""
    b, m, n, h, hk, d, half = CASE[:7]
    q, k, qw, kw, q_pos, k_pos, inv = make(CASE, gpu)
    dq_out, dk_out = torch.randn_like(q), torch.randn_like(k)
    shape = N.int64_array([b, m, n, h, hk, d])
    strides = N.int64_array([*q.stride()[:3], *k.stride()[:3], 0, 0])
    size = N.lib().bmx_qk_norm_rope_workspace_bytes(d)
    ws = torch.empty(size, device=gpu, dtype=torch.uint8)

    def grads(wanted):
        out = [torch.full_like(t, 7.0) for t in (q, k, qw, kw)]
        ptr = [t.data_ptr() if w else None for t, w in zip(out, wanted)]
        dy = [t.data_ptr() if ptr[i] or ptr[i + 2] else None for i, t in enumerate((dq_out, dk_out))]
        N.call("bmx_qk_norm_rope_bwd", q.data_ptr(), k.data_ptr(), N.BF16, shape, strides, qw.data_ptr(), kw.data_ptr(), N.BF16,
               q_pos.data_ptr(), k_pos.data_ptr(), 1, inv.data_ptr(), 1, half, 0, 1e-6, *dy, *ptr, ws.data_ptr(), size,
               torch.cuda.current_stream().cuda_stream)
        return out

    whole = grads((True,) * 4)
    for wanted in itertools.product((True, False), repeat=4):
        for w, some, every in zip(wanted, grads(wanted), whole):
            assert torch.equal(some, every if w else torch.full_like(every, 7.0)), wanted
