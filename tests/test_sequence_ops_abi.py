"""Argument checks of the sequence operators' C entry points: every rejection
happens before a launch, so they run without a GPU.  And the bucket
thresholds against their definition."""

import ctypes

import pytest

from boltz_lumi_amd import _native as N
from boltz_lumi_amd import ops


@pytest.fixture(scope="module")
def lib():
    if not N.lib_path().exists():
        pytest.skip("libbmx.so not built")
    return N.lib()


FAKE, ODD = ctypes.c_void_p(256), ctypes.c_void_p(260)


def refused(lib, rc, text):
    return rc == N.BMX_EINVAL and text in lib.bmx_last_error()


def test_qk_norm_rope_rejects_bad_arguments(lib):
    def fwd(q=FAKE, dtype=1, shape=(2, 5, 7, 4, 2, 64), strides=(1280, 256, 64, 896, 128, 64, 0, 0), qw=FAKE, wd=0,
            half=32, eps=1e-6, out=FAKE, k_pos=FAKE, inv=FAKE):
        return lib.bmx_qk_norm_rope_fwd(q, FAKE, dtype, N.int64_array(shape), N.int64_array(strides), qw, FAKE, wd, FAKE,
                                        k_pos, 1, inv, 1, half, 0, eps, out, FAKE, None)

    assert refused(lib, fwd(dtype=2), b"dtype") and refused(lib, fwd(wd=3), b"weight dtype")
    assert refused(lib, fwd(shape=(2, 5, 7, 4, 2, 60)), b"multiple of 8")
    assert refused(lib, fwd(shape=(2, 5, 7, 4, 2, 264)), b"[8, 256]")
    assert refused(lib, fwd(shape=(2, -1, 7, 4, 2, 64)), b"negative size")
    assert refused(lib, fwd(half=36), b"half the head dim") and refused(lib, fwd(half=2), b"multiple of 4")
    assert refused(lib, fwd(eps=0.0), b"eps") and refused(lib, fwd(inv=None), b"inv_freq")
    assert refused(lib, fwd(strides=(1280, 258, 64, 896, 128, 64, 0, 0)), b"strides")
    assert refused(lib, fwd(q=None), b"null pointer") and refused(lib, fwd(k_pos=None), b"null pointer")
    assert refused(lib, fwd(q=ODD), b"aligned") and refused(lib, fwd(qw=ODD), b"aligned")
    assert fwd(shape=(0, 5, 7, 4, 2, 64), q=None, out=None) == N.BMX_OK
    need = lib.bmx_qk_norm_rope_workspace_bytes(64)
    assert need == 2 * 1024 * 64 * 4 and lib.bmx_qk_norm_rope_workspace_bytes(0) == 0

    def bwd(qw=FAKE, ws=FAKE, size=need, dy=FAKE):
        return lib.bmx_qk_norm_rope_bwd(FAKE, FAKE, 1, N.int64_array((2, 5, 7, 4, 2, 64)),
                                        N.int64_array((1280, 256, 64, 896, 128, 64, 0, 0)), qw, FAKE, 0, FAKE, FAKE, 1,
                                        FAKE, 1, 32, 0, 1e-6, dy, FAKE, FAKE, FAKE, FAKE, FAKE, ws, size, None)

    assert refused(lib, bwd(size=need - 1), b"workspace") and refused(lib, bwd(ws=ODD), b"workspace")
    assert refused(lib, bwd(qw=None), b"absent weight") and refused(lib, bwd(dy=None), b"null pointer")


def test_relative_bias_rejects_bad_arguments(lib):
    edges = (ctypes.c_int32 * 15)(*ops._relative_thresholds(16, 8, 128))

    def fwd(table=FAKE, dtype=0, buckets=32, heads=4, batch=1, m=5, t=edges, count=15, both=1, out=FAKE):
        return lib.bmx_relative_bias_fwd(table, dtype, buckets, heads, FAKE, FAKE, 1, batch, m, 7, 0, 0, t, count, both,
                                         out, None)

    assert refused(lib, fwd(dtype=2), b"dtype") and refused(lib, fwd(buckets=300), b"[1, 256]")
    assert refused(lib, fwd(heads=0), b"heads") and refused(lib, fwd(m=-1), b"negative")
    assert refused(lib, fwd(both=0), b"this many buckets") and refused(lib, fwd(count=14), b"this many buckets")
    assert refused(lib, fwd(t=None), b"thresholds") and refused(lib, fwd(table=None), b"null pointer")
    assert refused(lib, fwd(t=(ctypes.c_int32 * 15)(*[1, 2, 2, 1] + [9] * 11)), b"rising")
    assert fwd(m=0, table=None, out=None) == N.BMX_OK
    need = lib.bmx_relative_bias_workspace_bytes(0, 32, 4, 1, 5, 7)
    assert need > 0 and lib.bmx_relative_bias_workspace_bytes(0, 32, 4, 1, 0, 7) == 0

    def bwd(dbias=FAKE, dtable=FAKE, ws=FAKE, size=need):
        return lib.bmx_relative_bias_bwd(dbias, 0, 32, 4, FAKE, FAKE, 1, 1, 5, 7, 0, 0, edges, 15, 1, dtable, ws, size, None)

    assert refused(lib, bwd(dbias=None), b"null pointer") and refused(lib, bwd(dtable=None), b"null pointer")
    assert refused(lib, bwd(size=need - 1), b"workspace") and refused(lib, bwd(ws=ODD), b"workspace")


@pytest.mark.parametrize("side,exact,top", [(2, 1, 128), (16, 8, 128), (33, 32, 32), (64, 20, 5000), (128, 3, 1 << 30),
                                            (128, 64, 65), (17, 1, 2)])
def test_thresholds(side, exact, top):
    """Threshold i is the least distance whose bucket is at least i."""
    edges = list(ops._relative_thresholds(side, exact, top))
    assert len(edges) == side - 1 and edges[:exact] == list(range(1, exact + 1)) and edges == sorted(edges)
    steps = side - exact
    for k, edge in enumerate(edges[exact:], 1):
        reach = exact ** (steps - k) * top ** k
        assert edge ** steps >= reach and (edge - 1) ** steps < reach


def test_cross_attention_rejects_bad_arguments(lib):
    b, m, n, h, hk, d = 2, 40, 50, 4, 2, 64
    good_shape = (b, m, n, h, hk, d)
    good_strides = (m * h * d, h * d, d, n * hk * d, hk * d, d, n * hk * d, hk * d, d, n, 0, m * n, n)
    need = lib.bmx_cross_attention_workspace_bytes(1, *good_shape)
    assert lib.bmx_cross_attention_workspace_bytes(1, b, 0, n, h, hk, d) == 0
    assert lib.bmx_cross_attention_workspace_bytes(1, 1, 1, 4096, 8, 2, d) > 0  # one query: split over the keys

    def fwd(q=FAKE, dtype=1, shape=good_shape, strides=good_strides, scale=0.1, out=FAKE, lo=FAKE, stats=FAKE, ws=FAKE,
            size=need):
        return lib.bmx_cross_attention_fwd(q, FAKE, FAKE, None, FAKE, dtype, N.int64_array(shape), N.int64_array(strides),
                                           scale, out, lo, stats, ws, size, None)

    assert refused(lib, fwd(dtype=2), b"dtype") and refused(lib, fwd(shape=(b, m, n, h, hk, 136)), b"[8, 128]")
    assert refused(lib, fwd(shape=(b, m, n, h, hk, 60)), b"multiple of 8")
    assert refused(lib, fwd(shape=(b, m, n, 5, hk, d)), b"multiple of the key heads")
    assert refused(lib, fwd(shape=(b, -1, n, h, hk, d)), b"negative size")
    assert refused(lib, fwd(scale=0.0), b"scale") and refused(lib, fwd(scale=float("nan")), b"scale")
    assert refused(lib, fwd(strides=(4, *good_strides[1:])), b"16 bytes")
    assert refused(lib, fwd(q=None), b"null pointer") and refused(lib, fwd(out=None), b"null pointer")
    assert refused(lib, fwd(q=ODD), b"16-byte aligned") and refused(lib, fwd(lo=ODD), b"16-byte aligned")
    assert refused(lib, fwd(stats=ODD), b"8-byte aligned")
    assert fwd(shape=(0, m, n, h, hk, d), q=None) == N.BMX_OK and fwd(shape=(b, 0, n, h, hk, d), q=None) == N.BMX_OK
    long = (1, 1, 4096, 8, 2, d)
    need_long = lib.bmx_cross_attention_workspace_bytes(1, *long)
    assert refused(lib, fwd(shape=long, size=need_long - 1), b"workspace")
    assert refused(lib, fwd(shape=long, ws=None, size=need_long), b"workspace")

    need_bwd = lib.bmx_cross_attention_bwd_workspace_bytes(b, m, n, h, hk, d)
    assert need_bwd == b * m * h * 4  # too few keys and queries to split
    assert lib.bmx_cross_attention_bwd_workspace_bytes(b, m, 0, h, hk, d) == 0
    assert lib.bmx_cross_attention_bwd_workspace_bytes(1, 128, 2048, 8, 8, d) >= 128 * 8 * 4 + 2 * 128 * 8 * d * 4

    def bwd(shape=good_shape, bias=FAKE, lo=FAKE, stats=FAKE, dout=FAKE, dq=FAKE, dbias=FAKE, steps=(0, m * n, n),
            ws=FAKE, size=need_bwd):
        return lib.bmx_cross_attention_bwd(FAKE, FAKE, FAKE, None, bias, 1, N.int64_array(shape),
                                           N.int64_array(good_strides), 0.1, FAKE, lo, stats, dout, dq, FAKE, FAKE, dbias,
                                           None if steps is None else N.int64_array(steps), ws, size, None)

    assert refused(lib, bwd(shape=(b, m, 0, h, hk, d)), b"empty") and refused(lib, bwd(lo=None), b"out_lo")
    assert refused(lib, bwd(bias=None), b"dbias needs") and refused(lib, bwd(steps=None), b"dbias needs")
    assert refused(lib, bwd(stats=None), b"null pointer") and refused(lib, bwd(dout=None), b"null pointer")
    assert refused(lib, bwd(dq=ODD), b"16-byte aligned") and refused(lib, bwd(stats=ODD), b"8-byte aligned")
    assert refused(lib, bwd(size=need_bwd - 1), b"workspace") and refused(lib, bwd(ws=ODD), b"workspace")
