"""Refusals of the sequence mixing operators: the C entry points' before any launch, the Python calls' plans, state
buffers, forward-mode derivatives and tracing.  Nothing here needs a GPU."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from boltz_lumi_amd import _native as N
from boltz_lumi_amd import ops

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lib():
    if not N.lib_path().exists():
        pytest.skip("libbmx.so not built")
    return N.lib()


FAKE, ODD = ctypes.c_void_p(256), ctypes.c_void_p(260)


def refused(lib, rc, text):
    return rc == N.BMX_EINVAL and text in lib.bmx_last_error()


def array(values):
    return N.int64_array(values)


def test_residual_norm_rejects_bad_arguments(lib):
    def fwd(x=FAKE, gate=FAKE, xd=0, d=1, shape=(2, 5, 64), strides=(320, 64, 320, 64, 320, 64), kind=1, yw=FAKE, wd=0, pre=1,
            eps=1e-6, r=FAKE, h=FAKE):
        return lib.bmx_residual_norm_fwd(x, FAKE, gate, xd, d, array(shape), array(strides), kind, yw, FAKE, FAKE, wd, 1, pre,
                                         eps, r, h, None)

    assert refused(lib, fwd(xd=2), b"fp32 or bf16") and refused(lib, fwd(xd=1, d=0), b"fp32 x where y is fp32")
    assert refused(lib, fwd(wd=2), b"weight dtype") and refused(lib, fwd(kind=3), b"gate")
    assert refused(lib, fwd(shape=(2, 5, 60)), b"multiple of 8") and refused(lib, fwd(shape=(2, 5, 8200)), b"8192")
    assert refused(lib, fwd(shape=(-1, 5, 64)), b"negative") and refused(lib, fwd(shape=(1 << 20, 1 << 20, 64)), b"2^31 rows")
    assert refused(lib, fwd(strides=(320, 60, 320, 64, 320, 64)), b"strides") and refused(lib, fwd(eps=0.0), b"eps")
    assert refused(lib, fwd(x=None), b"null pointer") and refused(lib, fwd(h=None), b"null pointer")
    assert refused(lib, fwd(gate=None), b"null pointer") and refused(lib, fwd(x=ODD), b"aligned")
    assert refused(lib, fwd(yw=ODD), b"aligned")
    assert fwd(shape=(0, 5, 64), x=None, r=None) == N.BMX_OK
    need = lib.bmx_residual_norm_workspace_bytes(2, 5, 64, 2)
    assert need > 0 and lib.bmx_residual_norm_workspace_bytes(0, 5, 64, 1) == 0

    def bwd(kind=2, yw=FAKE, dgate=FAKE, ws=FAKE, size=need, rows=5):
        return lib.bmx_residual_norm_bwd(FAKE, FAKE, FAKE, 0, 1, array((2, rows, 64)), array((320, 64) * 3), kind, yw, FAKE,
                                         FAKE, 0, 1, 1, 1e-6, FAKE, FAKE, FAKE, FAKE, dgate, FAKE, FAKE, FAKE, ws, size, None)

    assert refused(lib, bwd(size=need - 1), b"workspace") and refused(lib, bwd(ws=ODD), b"workspace")
    assert refused(lib, bwd(kind=0), b"absent gate") and refused(lib, bwd(yw=None), b"absent weight")
    assert refused(lib, bwd(dgate=ODD), b"aligned") and refused(lib, bwd(rows=0), b"rows")


def test_causal_conv_rejects_bad_arguments(lib):
    def fwd(x=FAKE, d=1, shape=(2, 5, 64, 4), strides=(320, 64), w=FAKE, wd=0, bd=0, state=FAKE, y=FAKE, out=FAKE):
        return lib.bmx_causal_conv_fwd(x, d, array(shape), array(strides), w, wd, FAKE, bd, state, FAKE, 1, 1, y, out, None)

    assert refused(lib, fwd(d=2), b"dtype") and refused(lib, fwd(wd=2), b"dtypes") and refused(lib, fwd(bd=5), b"dtypes")
    assert refused(lib, fwd(shape=(2, 5, 60, 4)), b"multiple of 8") and refused(lib, fwd(shape=(2, 5, 1 << 20, 4)), b"2^20")
    assert refused(lib, fwd(shape=(2, 5, 64, 1)), b"width") and refused(lib, fwd(shape=(2, 5, 64, 5)), b"width")
    assert refused(lib, fwd(shape=(2, -5, 64, 4)), b"negative")
    assert refused(lib, fwd(shape=(1 << 16, 1 << 16, 64, 4)), b"2^31 rows")
    assert refused(lib, fwd(strides=(320, 60)), b"strides") and refused(lib, fwd(x=None), b"null pointer")
    assert refused(lib, fwd(w=None), b"null pointer") and refused(lib, fwd(y=None), b"null pointer")
    assert refused(lib, fwd(state=ODD), b"aligned") and refused(lib, fwd(out=ODD), b"aligned")
    assert refused(lib, fwd(shape=(2, 0, 64, 4)), b"no tokens")
    assert fwd(shape=(0, 5, 64, 4), x=None, y=None) == N.BMX_OK
    assert fwd(shape=(2, 0, 64, 4), x=None, y=None, out=None) == N.BMX_OK
    need = lib.bmx_causal_conv_workspace_bytes(2, 5, 64, 4)
    assert need > 0 and lib.bmx_causal_conv_workspace_bytes(2, 0, 64, 4) == 0

    def bwd(bias=FAKE, state=FAKE, dx=FAKE, ws=FAKE, size=need, rows=5):
        return lib.bmx_causal_conv_bwd(FAKE, 1, array((2, rows, 64, 4)), array((320, 64)), FAKE, 0, bias, 0, state, None, 0, 1,
                                       FAKE, FAKE, dx, FAKE, FAKE, FAKE, ws, size, None)

    assert refused(lib, bwd(size=need - 1), b"workspace") and refused(lib, bwd(ws=ODD), b"workspace")
    assert refused(lib, bwd(bias=None), b"absent") and refused(lib, bwd(state=None), b"absent")
    assert refused(lib, bwd(dx=ODD), b"aligned") and refused(lib, bwd(rows=0), b"rows")


def test_selective_scan_rejects_bad_arguments(lib):
    steps = (320, 64) * 3 + (80, 16, 16) * 2

    def fwd(u=FAKE, d=1, shape=(2, 5, 64, 16, 1), strides=steps, A=FAKE, z=FAKE, state=FAKE, out=FAKE, last=FAKE, raw=None,
            ws=FAKE, size=1 << 30):
        return lib.bmx_selective_scan_fwd(u, FAKE, A, FAKE, FAKE, FAKE, z, FAKE, state, FAKE, d, 1, array(shape),
                                          array(strides), 1, out, last, None, raw, ws, size, None)

    assert refused(lib, fwd(d=2), b"dtype") and refused(lib, fwd(shape=(2, 5, 64, 12, 1)), b"states")
    assert refused(lib, fwd(shape=(2, 5, 60, 16, 1)), b"multiple of 8")
    assert refused(lib, fwd(shape=(2, 5, 72, 16, 2)), b"multiple of 8 per group")
    assert refused(lib, fwd(shape=(2, 5, 64, 16, 0)), b"per group") and refused(lib, fwd(shape=(2, 5, 1 << 20, 16, 1)), b"2^20")
    assert refused(lib, fwd(shape=(2, -1, 64, 16, 1)), b"negative")
    assert refused(lib, fwd(shape=(1 << 16, 1 << 16, 64, 16, 1)), b"2^31 rows")
    assert refused(lib, fwd(strides=(320, 62, *steps[2:])), b"strides") and refused(lib, fwd(u=None), b"null pointer")
    assert refused(lib, fwd(A=None), b"null pointer") and refused(lib, fwd(out=None), b"out")
    assert refused(lib, fwd(state=ODD), b"aligned") and refused(lib, fwd(u=ODD), b"aligned")
    assert refused(lib, fwd(z=None, raw=FAKE), b"raw") and refused(lib, fwd(shape=(2, 0, 64, 16, 1)), b"no tokens")
    long = (1, 4096, 64, 16, 1)
    need = lib.bmx_selective_scan_workspace_bytes(*long)
    assert need > 0 and refused(lib, fwd(shape=long, size=need - 1), b"workspace")
    assert refused(lib, fwd(shape=long, ws=None), b"workspace")
    assert fwd(shape=(0, 5, 64, 16, 1), u=None, out=None) == N.BMX_OK
    assert lib.bmx_selective_scan_workspace_bytes(1, 1, 64, 16, 1) == 0
    assert lib.bmx_selective_scan_saved_bytes(2, 33, 64, 16) == 2 * 3 * 64 * 16 * 4
    size = lib.bmx_selective_scan_bwd_workspace_bytes(2, 5, 64, 16, 1)

    def bwd(D=FAKE, z=FAKE, bias=FAKE, saved=FAKE, raw=FAKE, du=FAKE, ws=FAKE, size=size, rows=5):
        return lib.bmx_selective_scan_bwd(FAKE, FAKE, FAKE, FAKE, FAKE, D, z, bias, None, 1, 0, array((2, rows, 64, 16, 1)),
                                          array(steps), 1, saved, raw, FAKE, None, du, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                          FAKE, FAKE, ws, size, None)

    assert refused(lib, bwd(size=size - 1), b"workspace") and refused(lib, bwd(ws=ODD), b"workspace")
    assert refused(lib, bwd(D=None), b"absent") and refused(lib, bwd(z=None), b"absent")
    assert refused(lib, bwd(bias=None), b"absent") and refused(lib, bwd(saved=None), b"null pointer")
    assert refused(lib, bwd(raw=None), b"null pointer") and refused(lib, bwd(du=ODD), b"aligned")
    assert refused(lib, bwd(rows=0), b"rows")
    assert refused(lib, bwd(D=ODD), b"aligned") and refused(lib, bwd(bias=ODD), b"aligned")


def layouts(*tensors):
    return [ops._layout(t) for t in tensors]


def e(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype)


@pytest.mark.parametrize("change,text", [
    (dict(y=e(2, 5, 32)), "one shape"), (dict(x=e(2, 5, 64), y=e(2, 5, 64, dtype=FP32)), "fp32 y"),
    (dict(x=e(2, 5, 60), y=e(2, 5, 60)), "multiple of 8"), (dict(gate=e(2, 4, 64)), "gate"), (dict(gate=e(1, 1, 64)), "gate"),
    (dict(gate=e(2, 5, 64, dtype=FP32)), "gate"), (dict(scale=e(32)), "weights"), (dict(scale=e(64)), "share a dtype"),
    (dict(weight=e(64, dtype=torch.float16)), "weights"), (dict(post=False), "y_weight"), (dict(pre=False), "weight needs"),
    (dict(x=e(2, 5, 64, dtype=torch.float16)), "dtype")])
def test_frame_plan_refuses(change, text):
    v = dict(x=e(2, 5, 64), y=e(2, 5, 64), gate=e(2, 5, 64), y_weight=e(64, dtype=FP32), scale=e(64, dtype=FP32),
             weight=e(64, dtype=FP32), post=True, pre=True)
    v.update(change)
    post, pre = v.pop("post"), v.pop("pre")
    with pytest.raises(RuntimeError, match=text):
        ops._frame_plan(*layouts(*v.values()), post, pre)


@pytest.mark.parametrize("change,text", [
    (dict(x=e(2, 5, 60)), "multiple of 8"), (dict(weight=e(64, 5)), "width"), (dict(weight=e(64, 1)), "width"),
    (dict(weight=e(32, 4)), "width"), (dict(bias=e(32)), "bias"), (dict(state=e(2, 2, 64)), "state"),
    (dict(state=e(2, 3, 64, dtype=FP32)), "state"), (dict(lengths=e(3, dtype=torch.int64)), "lengths"),
    (dict(lengths=e(2, dtype=FP32)), "lengths"), (dict(weight=e(64, 4, dtype=torch.float16)), "weight and bias")])
def test_conv_plan_refuses(change, text):
    v = dict(x=e(2, 5, 64), weight=e(64, 4), bias=e(64), state=e(2, 3, 64), lengths=e(2, dtype=torch.int32))
    v.update(change)
    with pytest.raises(RuntimeError, match=text):
        ops._conv_plan(*layouts(*v.values()), 1)


@pytest.mark.parametrize("change,text", [
    (dict(dt=e(2, 5, 32)), "dt and z"), (dict(z=e(2, 5, 64, dtype=FP32)), "dt and z"), (dict(B=e(2, 5, 1, 8)), "B and C"),
    (dict(A=e(64, 12, dtype=FP32), B=e(2, 5, 1, 12), C=e(2, 5, 1, 12)), "states must"), (dict(A=e(64, 16)), "A "),
    (dict(A=e(32, 16, dtype=FP32)), "A "), (dict(B=e(2, 5, 3, 16), C=e(2, 5, 3, 16)), "multiple of 8"),
    (dict(D=e(64)), "D and dt_bias"), (dict(dt_bias=e(32, dtype=FP32)), "D and dt_bias"), (dict(state=e(2, 64, 16)), "state"),
    (dict(state=e(2, 64, 8, dtype=FP32)), "state"), (dict(lengths=e(2, 1, dtype=torch.int64)), "lengths")])
def test_scan_plan_refuses(change, text):
    v = dict(u=e(2, 5, 64), dt=e(2, 5, 64), A=e(64, 16, dtype=FP32), B=e(2, 5, 1, 16), C=e(2, 5, 1, 16), D=e(64, dtype=FP32),
             z=e(2, 5, 64), dt_bias=e(64, dtype=FP32), state=e(2, 64, 16, dtype=FP32), lengths=e(2, dtype=torch.int64))
    v.update(change)
    with pytest.raises(RuntimeError, match=text):
        ops._scan_plan(*layouts(*v.values()), 1)


def test_state_buffers():
    """A buffer for the last state may be the first one, and nothing else that the call reads."""
    memory = torch.zeros(4, 3, 64, dtype=BF16)
    state, x = memory[:2], torch.zeros(2, 5, 64, dtype=BF16)

    def check(out, state=state, x=x, grad=False):
        plan = ops._conv_plan(*layouts(x, e(64, 4), None, state, None), 1)
        ops._check_state_out(out, plan, BF16, state, (x, None, None, None), grad)

    check(state)
    check(memory[2:])
    check(state.view(2, 3, 64))
    check(memory[1:3], x=memory.flatten()[:128].view(1, 2, 64).expand(2, 2, 64), state=None)  # in front of it
    for out, text in ((memory[1:3], "shares memory"), (torch.zeros(2, 3, 64), "dense"), (torch.zeros(2, 3, 128, dtype=BF16)
                      [..., :64], "dense"), (memory.flatten()[4:4 + 384].view(2, 3, 64), "aligned"),
                      (torch.zeros(1, 3, 64, dtype=BF16).expand(2, 3, 64), "dense")):
        with pytest.raises(RuntimeError, match=text):
            check(out)
    with pytest.raises(RuntimeError, match="shares memory"):
        check(memory[:2], state=None, x=memory[1:].flatten()[:256].view(2, 2, 64))
    with pytest.raises(RuntimeError, match="shares memory"):
        check(memory[:2], state=None, x=memory[:2])  # the inputs themselves are not the state
    with pytest.raises(RuntimeError, match="return_state"):
        check(state, grad=True)


def norm(x):
    return ops.residual_norm(x, x)[0]


def norm_weight(x):
    return ops.residual_norm(x.detach(), x.detach(), weight=x[0, 0])[0]


def conv(x):
    return ops.causal_conv(x, x[0, :4].T.contiguous())


def conv_state(x):
    return ops.causal_conv(x.detach(), x[0, :4].detach().T.contiguous(), state=x[:, :3])


def scan(x):
    return ops.selective_scan(x, x, x[0, :, None].expand(8, 8, 8)[0], x[:, :, None], x[:, :, None])


OPERATORS = [norm, norm_weight, conv, conv_state, scan]


@pytest.mark.parametrize("operator", OPERATORS)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(operator, grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x = forward_ad.make_dual(torch.randn(1, 8, 8), torch.ones(1, 8, 8))
        with pytest.raises(RuntimeError, match="forward-mode"):
            operator(x)


@pytest.mark.parametrize("operator", OPERATORS)
def test_tracing_is_refused(operator):
    x = torch.randn(1, 8, 8)
    with pytest.raises(RuntimeError, match="tracing"):
        make_fx(operator)(x)
    with pytest.raises(RuntimeError, match="tracing"):
        torch.jit.trace(operator, x)


@pytest.mark.parametrize("operator", OPERATORS)
def test_cpu_tensors_are_refused(operator):
    with pytest.raises(RuntimeError, match="CUDA"):
        operator(torch.randn(1, 8, 8))

