"""Argument checks of the operators on a paged cache at their edges (CPU: they come before any device
access)."""

import ctypes as C

import pytest

from kvcache_manager import _native

P16 = 1 << 20  # an aligned address that is never read
S2, S3 = C.c_int64 * 2, C.c_int64 * 3


def cache(**change):
    """2 requests of 2 pages of 16 tokens, 2 KV heads of 64."""
    c = _native.PagedCache(P16, P16, S3(4096, 2048, 128), S3(4096, 2048, 128), P16, 4, 2, 16, 64, 2, 2, _native.DTYPE_BF16, 1.0, 1.0)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def error(rc):
    assert rc == _native.E_INVAL
    return _native.load().kvs_last_error().decode()


@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
def test_scales_without_a_reciprocal(name):
    """The fill multiplies by 1 / scale: below 2^-128 that is infinite, and zeros would become NaN."""
    lib = _native.load()
    for scale, refused in ((1e-39, True), (2.0**-149, True), (2.0**-128, True), (2.0**-127, False), (3e38, False)):
        rows = _native.DecodeRows(q_heads=3)  # refused after the cache was found right
        message = error(lib.kvs_paged_decode_attention(C.byref(cache(dtype=2, **{name: scale})), C.byref(rows), None))
        assert ("reciprocal" in message) == refused and ("multiple of the KV heads" in message) != refused, (scale, message)
