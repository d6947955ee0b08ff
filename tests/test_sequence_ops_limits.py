"""Sizes past what the sequence operators' launches take are refused by name, before a launch (no GPU needed)."""

import ctypes

import pytest

from boltz_lumi_amd import _native as N


@pytest.fixture(scope="module")
def lib():
    if not N.lib_path().exists():
        pytest.skip("libbmx.so not built")
    return N.lib()


FAKE = ctypes.c_void_p(256)


def refused(lib, rc, text):
    return rc == N.BMX_EINVAL and text in lib.bmx_last_error()


def test_norm_rope_rows(lib):
    """256 rows of 8 channels a block, below 2^24 blocks."""
    def fwd(tokens):
        return lib.bmx_qk_norm_rope_fwd(FAKE, None, N.BF16, N.int64_array((1, tokens, 0, 1, 0, 8)),
                                        N.int64_array((0, 8, 8, 0, 0, 0, 0, 0)), None, None, N.BF16, None, None, 1, None, 1, 0,
                                        0, 1e-6, FAKE, None, None)

    assert refused(lib, fwd(((1 << 24) - 1) * 256 + 1), b"too many rows") and refused(lib, fwd(1 << 36), b"too many rows")


def test_attention_blocks(lib):
    shape = (1 << 29, 1, 2, 4, 4, 8)
    strides = N.int64_array((32, 32, 8, 64, 32, 8, 64, 32, 8, 0, 0, 0, 0))
    rc = lib.bmx_cross_attention_fwd(FAKE, FAKE, FAKE, None, None, N.BF16, N.int64_array(shape), strides, 0.1, FAKE, None,
                                     None, None, 0, None)
    assert refused(lib, rc, b"too many blocks")
    size = lib.bmx_cross_attention_bwd_workspace_bytes(*shape)
    rc = lib.bmx_cross_attention_bwd(FAKE, FAKE, FAKE, None, None, N.BF16, N.int64_array(shape), strides, 0.1, FAKE, FAKE, FAKE,
                                     FAKE, FAKE, None, None, None, None, FAKE, size, None)
    assert refused(lib, rc, b"too many blocks")


def test_table_gradient_blocks(lib):
    edges = (ctypes.c_int32 * 1)(1)
    batch, heads = 1 << 27, 16
    size = lib.bmx_relative_bias_workspace_bytes(N.F32, 4, heads, batch, 1, 1)
    rc = lib.bmx_relative_bias_bwd(FAKE, N.F32, 4, heads, FAKE, FAKE, 1, batch, 1, 1, 1, 1, edges, 1, 1, FAKE, FAKE, size, None)
    assert refused(lib, rc, b"too many elements")


def test_attention_scale(lib):
    """A scale that fp32 flushes to zero, or whose product with log2(e) it cannot hold, made every result NaN."""
    def fwd(scale):
        return lib.bmx_cross_attention_fwd(FAKE, FAKE, FAKE, None, None, N.BF16, N.int64_array((1, 0, 2, 1, 1, 8)),
                                           N.int64_array((8, 8, 8, 16, 8, 8, 16, 8, 8, 0, 0, 0, 0)), scale, FAKE, None, None,
                                           None, 0, None)

    for scale in (1e-40, 2.0 ** -127, 3e38, -1.0):
        assert refused(lib, fwd(scale), b"scale")
    for scale in (2.0 ** -126, 2.0 ** 127, 0.125):
        assert fwd(scale) == N.BMX_OK  # without queries nothing is launched


def test_norm_rope_eps(lib):
    """An eps that fp32 flushes to zero made rows of zeros NaN."""
    def fwd(eps):
        return lib.bmx_qk_norm_rope_fwd(FAKE, None, N.BF16, N.int64_array((1, 0, 0, 1, 0, 8)),
                                        N.int64_array((0, 8, 8, 0, 0, 0, 0, 0)), None, None, N.BF16, None, None, 1, None, 1, 0,
                                        0, eps, FAKE, None, None)

    assert all(refused(lib, fwd(eps), b"eps") for eps in (1e-40, 2.0 ** -127, -1e-6, float("nan")))
    assert fwd(2.0 ** -126) == N.BMX_OK and fwd(1e-6) == N.BMX_OK
