"""What the tests of the sequence mixing operators share: inputs from a seed and the comparison with the oracle."""

import torch

FP32, BF16 = torch.float32, torch.bfloat16


def randn(g, *shape, dtype=FP32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift).to(dtype)


def fp64(t):
    return None if t is None else t.detach().cpu().double()


def leaf(t, device):
    return None if t is None else t.to(device).requires_grad_()


def assert_close(name, got, want, size, roundings):
    """``got`` within its type's rounding of the exact result (half a step of it) and ``roundings`` roundings of 2^-24
    relative to ``size``, the magnitudes of the terms that it sums.  A result that is rounded to 16 bits may sit on the
    other side of a rounding border, a whole step away from the exact value's: the half step is of got or want, whichever
    is larger."""
    if want is None:
        assert got is None, name
        return
    assert tuple(got.shape) == tuple(want.shape), (name, got.shape, want.shape)
    got = got.detach()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != FP32 else 2.0 ** -24
    g = got.cpu().double()
    assert torch.isfinite(g).all(), f"{name}: not finite"
    limit = half * torch.maximum(g.abs(), want.abs()) + roundings * 2.0 ** -24 * size + 2.0 ** -120
    over = ((g - want).abs() / limit)
    assert not over.numel() or over.max() <= 1, (
        f"{name}: {over.max():.3g} of what it may be off at {over.argmax()}: {g.flatten()[over.argmax()]} for "
        f"{want.flatten()[over.argmax()]}")
