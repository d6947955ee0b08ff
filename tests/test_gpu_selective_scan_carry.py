"""ops.selective_scan where its states are carried by one thread each (65536 states of a batch and more) and where a
block of the gradient takes two tiles of tokens: ragged lengths, a first state, gradients of the last one, and decays so
slow that what is carried matters to the end, against the oracle in fp64.

Tolerances as in the other tests of the scan: half a step of the result's type, and roundings of 2^-24 relative to the
magnitudes that a value is made of: 8 a token that a term lives for (its decay's exponent is below 1 here), 96 for the
rest, one a row for a sum over rows.  A state or gradient that came to a chunk without its first part would be off by a
tenth of its size, hundreds of times as much."""

import pytest
import torch

from boltz_lumi_amd import ops
from oracle import mixing
from mixing_cases import BF16, FP32, assert_close, leaf, randn

pytestmark = pytest.mark.gpu

NAMES = ["out", "state", "du", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dstate"]


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def check(b, t, c, n, groups, dtype, lengths, gpu, decay=0.02):
    g = torch.Generator().manual_seed(b * t + c)
    u, z, dt = (randn(g, b, t, c, dtype=dtype) for _ in range(3))
    B, C = (randn(g, b, t, groups, n, dtype=dtype) for _ in range(2))
    inputs = [u, dt, -decay * (randn(g, c, n).abs() + 0.1), B, C, randn(g, c), z, randn(g, c, scale=0.5, shift=-2.0),
              randn(g, b, c, n)]
    back = [randn(g, b, t, c, dtype=dtype), randn(g, b, c, n)]
    leaves = [leaf(v, gpu) for v in inputs]
    out = ops.selective_scan(*leaves[:8], state=leaves[8], lengths=torch.tensor(lengths, device=gpu), return_state=True)
    grads = torch.autograd.grad(out, leaves, [v.to(gpu) for v in back])
    with torch.no_grad(), torch.device(gpu):  # the oracle's thousands of small steps, in fp64 on the device
        results, sizes = mixing.selective_scan(*(v.to(gpu).double() for v in inputs), lengths, True,
                                               *(v.to(gpu).double() for v in back))
    for name, got, want, size in zip(NAMES, (*out, *grads), results, sizes):
        rows = b * t if name in ("dA", "dD", "ddt_bias") else c if name in ("dB", "dC") else 0
        assert_close(name, got, want.cpu(), size.cpu(), 96 + 8 * max(lengths) + rows)


@pytest.mark.parametrize("c", [1016, 1024])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_around_65536_states(gpu, c, dtype):
    """Ten chunks, more than one load of them, by runs of chunks and by one thread a state."""
    check(4, 300, c, 16, 1, dtype, [300, 299, 161, 40], gpu)


def test_many_states(gpu):
    check(4, 300, 1536, 16, 1, BF16, [300, 257, 32, 0], gpu)


@pytest.mark.parametrize("n", [8, 16, 32, 64])
@pytest.mark.parametrize("t", [100, 130])
def test_two_tiles_a_range(gpu, n, t):
    """32 groups of 8 channels, 12 sequences: 1536 tiles and more, so two a block; lengths that end in either of them and
    between, and (130 tokens) a last range of one tile."""
    lengths = [t, t - 1, 97, 96, 95, 65, 64, 63, 33, 17, 1, 0]
    check(12, t, 256, n, 32, FP32, lengths, gpu)


def test_two_tiles_a_range_of_64_states(gpu):
    """Two blocks a compute unit, so from 1024 tiles on."""
    check(8, 100, 256, 64, 32, FP32, [100, 99, 97, 96, 64, 33, 1, 0], gpu)


def test_two_tiles_a_range_of_several_spans(gpu):
    """Maps' gradients added over spans of channels, of two groups."""
    check(64, 130, 512, 16, 2, BF16, [130 - 2 * i for i in range(64)], gpu)
