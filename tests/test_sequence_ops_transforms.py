"""Forward-mode derivatives and tracers do not see a native launch: the sequence
operators refuse them instead of dropping tangents or recording empty tensors.
The refusal comes before anything looks at a device, so it is tested on the CPU."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from boltz_lumi_amd import ops


def attention(x):
    return ops.cross_attention(x, x, x)


def attention_bias(x):
    bias = x[:, :, :1].transpose(1, 2).expand(1, 1, 5, 8)[..., :5]
    return ops.cross_attention(x.detach(), x.detach(), x.detach(), None, bias)


def norm_rope(x):
    return ops.qk_norm_rope(x, None, None, None, None, None, None)[0]


def norm_rope_weight(x):
    return ops.qk_norm_rope(x.detach(), None, x[0, 0, 0], None, None, None, None)[0]


def relative(x):
    return ops.relative_bias(x[0, :4, 0], torch.arange(3), torch.arange(3), exact=1)


OPERATORS = [attention, attention_bias, norm_rope, norm_rope_weight, relative]


@pytest.mark.parametrize("operator", OPERATORS)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(operator, grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x = forward_ad.make_dual(torch.randn(1, 5, 1, 8), torch.ones(1, 5, 1, 8))
        with pytest.raises(RuntimeError, match="forward-mode"):
            operator(x)


@pytest.mark.parametrize("operator", OPERATORS)
def test_tracing_is_refused(operator):
    x = torch.randn(1, 5, 1, 8)
    with pytest.raises(RuntimeError, match="tracing"):
        make_fx(operator)(x)
    with pytest.raises(RuntimeError, match="tracing"):
        torch.jit.trace(operator, x)


@pytest.mark.parametrize("operator", OPERATORS)
def test_neither_without_them(operator):
    """A level that the tensors have no tangent on is not refused; these are CPU tensors, which are."""
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="CUDA"):
            operator(torch.randn(1, 5, 1, 8))
