"""ops.causal_conv and its gradients against the oracle in fp64.

Tolerances: half a step of the result's type, and roundings of 2^-24 relative to the magnitudes that a value is made of:
at most four products and their sum, a sigmoid of the hardware exponential and reciprocal (4) and its slope, the taps
again: under 48.  A weight's sum over rows adds at most one a row."""

import pytest
import torch

from boltz_lumi_amd import ops
from oracle import mixing
from mixing_cases import BF16, FP32, assert_close, fp64, leaf, randn

pytestmark = pytest.mark.gpu

NAMES = ["y", "state", "dx", "dweight", "dbias", "dstate"]


def make(b, t, c, width, dtype, w_dtype=FP32, bias=True, state=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    inputs = [randn(g, b, t, c, dtype=dtype), randn(g, c, width, dtype=w_dtype, scale=0.6),
              randn(g, c, dtype=w_dtype, scale=0.2) if bias else None,
              randn(g, b, width - 1, c, dtype=dtype) if state else None]
    return inputs, [randn(g, b, t, c, dtype=dtype), randn(g, b, width - 1, c, dtype=dtype)]


def check(inputs, back, gpu, lengths=None, silu=True, view=lambda t: t, index=torch.int64):
    leaves = [leaf(t, gpu) for t in inputs]
    b, t = inputs[0].shape[:2]
    on_gpu = None if lengths is None else torch.tensor(lengths, device=gpu, dtype=index)
    made = ops.causal_conv(view(leaves[0]), leaves[1], leaves[2], state=leaves[3], lengths=on_gpu, silu=silu,
                           return_state=True)
    wanted = [x for x in leaves if x is not None]
    grads = iter(torch.autograd.grad(made, wanted, [x.to(gpu) for x in back]))
    got = [*made, *(None if x is None else next(grads) for x in leaves)]
    ends = [t] * b if lengths is None else [min(max(n, 0), t) for n in lengths]
    with torch.no_grad():
        results, sizes = mixing.causal_conv(*map(fp64, inputs), ends, silu, *map(fp64, back))
    for name, a, w, size in zip(NAMES, got, results, sizes):
        assert_close(name, a, w, size, 48 + (b * t if name in ("dweight", "dbias") else 0))
    return got


@pytest.mark.parametrize("t", [1, 2, 3, 4, 5, 8, 15, 16, 17, 63, 64, 65, 130])
@pytest.mark.parametrize("width", [2, 3, 4])
def test_lengths_of_tokens(gpu, t, width):
    check(*make(2, t, 24, width, BF16, seed=t), gpu)


@pytest.mark.parametrize("c", [8, 16, 128, 136, 256, 264, 520])
@pytest.mark.parametrize("dtype,w_dtype", [(BF16, FP32), (BF16, BF16), (FP32, FP32)])
def test_channels_and_types(gpu, c, dtype, w_dtype):
    check(*make(3, 21, c, 4, dtype, w_dtype, seed=c), gpu)


@pytest.mark.parametrize("bias,state", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("silu", [True, False])
def test_absent_parts(gpu, bias, state, silu):
    check(*make(2, 19, 40, 3, FP32, bias=bias, state=state), gpu, silu=silu)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("width", [2, 4])
def test_ragged(gpu, index, width):
    """Lengths of nothing, of less than the taps, to the end and past both ends; rows behind them are NaN and stay unseen."""
    lengths = [0, 1, 2, 3, 18, 33, 34, 99, -5]
    inputs, back = make(9, 34, 16, width, BF16)
    for i, n in enumerate(lengths):
        inputs[0][i, max(n, 0):] = float("nan")
        back[0][i, max(n, 0):] = float("nan")
    clean = [torch.nan_to_num(t) for t in (inputs[0], back[0])]
    got = check(inputs, back, gpu, lengths, index=index)
    want, _ = mixing.causal_conv(fp64(clean[0]), *map(fp64, inputs[1:]), [min(max(n, 0), 34) for n in lengths], True,
                                 fp64(clean[1]), fp64(back[1]))
    for i, n in enumerate(lengths):
        assert not got[0][i, max(n, 0):].any() and not got[2][i, max(n, 0):].any()
    assert torch.equal(got[1].cpu().double(), want[1])


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides(gpu, dtype):
    inputs, back = make(3, 9, 32, 4, dtype)

    def slices(t):
        wide = torch.full((3, 9, 96), float("nan"), device=t.device, dtype=t.dtype)
        wide[..., 32:64] = t
        return wide[..., 32:64]

    for view in (slices, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)):
        check(inputs, back, gpu, view=view)


@pytest.mark.parametrize("parts", [[1] * 9, [4, 5], [2, 1, 3, 3], [8, 1]])
def test_parts_of_a_sequence(gpu, parts):
    """A sequence in parts, each from the state that the part before left, is the whole; in place too, bit for bit."""
    (x, w, b, first), _ = make(2, 9, 48, 4, BF16)
    x, w, b, first = (t.to(gpu) for t in (x, w, b, first))
    whole, last = ops.causal_conv(x, w, b, state=first, return_state=True)
    kept, moving, outs = first.clone(), first, []
    for part in x.split(parts, 1):
        y, moving = ops.causal_conv(part, w, b, state=moving, return_state=True)
        in_place = ops.causal_conv(part.contiguous(), w, b, state=kept, state_out=kept)
        outs.append(y)
        assert torch.equal(y, in_place) and torch.equal(moving, kept)
    assert torch.equal(torch.cat(outs, 1), whole) and torch.equal(moving, last)


def test_long_rows_and_many_runs(gpu):
    """Runs of 8 tokens a thread (from 2^19 runs of channels on), whose outputs are those of short calls, bit for bit."""
    (x, w, b, first), _ = make(2, 16400, 128, 4, BF16)
    x, w, b, first = (t.to(gpu) for t in (x, w, b, first))
    lengths = torch.tensor([16400, 4097], device=gpu)
    whole, last = ops.causal_conv(x, w, b, state=first, lengths=lengths, return_state=True)
    for at in (0, 7, 8, 4090, 16390):
        before = first if at == 0 else torch.cat([first, x], 1)[:, at:at + 3].contiguous()
        part = ops.causal_conv(x[:, at:at + 10], w, b, state=before)
        keep = (torch.arange(at, at + 10, device=gpu) < lengths[:, None])[..., None]
        assert torch.equal(torch.where(keep, part, torch.zeros_like(part)), whole[:, at:at + 10])
    assert torch.equal(last, torch.stack([x[0, -3:], x[1, 4094:4097]]))


def test_gradient_over_many_rows(gpu):
    """Partial sums of many blocks: ones times ones, which fp32 adds exactly."""
    x = torch.ones(3, 4100, 264, device=gpu, dtype=BF16)
    w = torch.zeros(264, 4, device=gpu, requires_grad=True)
    b = torch.zeros(264, device=gpu, requires_grad=True)
    y = ops.causal_conv(x, w, b, silu=False)
    dw, db = torch.autograd.grad(y, (w, b), torch.ones_like(y))
    assert torch.equal(db, torch.full_like(db, 3 * 4100))
    assert torch.equal(dw, torch.tensor([3 * (4100 - k) for k in (3, 2, 1, 0)], device=gpu).float().expand(264, 4))


@pytest.mark.parametrize("which", range(4))
def test_one_gradient(gpu, which):
    inputs, back = make(2, 33, 40, 3, BF16)
    for result in (0, 1):
        if result == 1 and which in (1, 2):
            continue  # the last inputs depend on neither
        leaves = [leaf(t, gpu) for t in inputs]
        made = ops.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], return_state=True)
        every = torch.autograd.grad(made[result], leaves, back[result].to(gpu), allow_unused=True)[which]
        leaves = [leaf(t, gpu) if i == which else t.to(gpu) for i, t in enumerate(inputs)]
        made = ops.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], return_state=True)
        alone, = torch.autograd.grad(made[result], leaves[which], back[result].to(gpu))
        assert torch.equal(alone, every)


def test_no_tokens(gpu):
    for b, t in ((0, 4), (2, 0)):
        inputs, _ = make(b, t, 16, 3, FP32)
        leaves = [leaf(x, gpu) for x in inputs]
        y, last = ops.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], return_state=True)
        assert y.shape == (b, t, 16) and torch.equal(last, leaves[3])
        dx, dw, db, ds = torch.autograd.grad((y, last), leaves, (y.detach(), torch.ones_like(last)))
        assert not dx.any() and not dw.any() and not db.any() and torch.equal(ds, torch.ones_like(last))
        kept = leaves[3].detach()
        ops.causal_conv(leaves[0].detach(), leaves[1].detach(), state=kept, state_out=kept)
        assert torch.equal(kept, leaves[3])


def test_state_out_is_seen_by_autograd(gpu):
    """A state that a gradient needs and that is written over afterwards is an error, not a wrong gradient."""
    (x, w, b, first), _ = make(1, 5, 16, 3, FP32)
    x, w, b, first = (t.to(gpu) for t in (x, w, b, first))
    y = ops.causal_conv(x, w.requires_grad_(), b, state=first)
    ops.causal_conv(x, w.detach(), b, state=first, state_out=first)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
