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


def test_evict_destination_that_starts_where_the_table_does():
    """The page table itself means in place. Other rows at its address are other tables, whose pages the
    call would read and write at once. (One request's row may be cut short behind `keep`.)"""
    lib, two = _native.load(), S2(512, 128)
    rows = lambda **kw: _native.EvictRows(**dict(dict(keep=8, w_len=32, wo_len=32, weights=P16, weights_out=P16, weights_strides=two,
                                                     weights_out_strides=two, dst_table=P16), **kw))
    call = lambda c, **kw: error(lib.kvs_evict_paged(C.byref(c), C.byref(rows(**kw)), None))
    assert "page_table itself" in call(cache(), dst_blocks=1)
    assert "must cover keep" in call(cache(batch=1), dst_blocks=1, keep=17)
    # taken as in place, then refused for their host addresses
    assert "must be on device" in call(cache(), dst_blocks=2) and "must be on device" in call(cache(batch=1), dst_blocks=1)


def test_attention_sums_that_overlap():
    """weights_out may be weights itself, not other rows at its address; strides of a dimension of one
    element do not matter."""
    lib = _native.load()
    rows = lambda **kw: _native.DecodeRows(**dict(dict(q=P16, out=P16, q_heads=4, scale=1.0, out_strides=S2(512, 128), weights=P16, weights_out=P16,
                                                       w_len=32, weights_strides=S2(64, 32), weights_out_strides=S2(64, 32)), **kw))
    attend = lambda c, **kw: error(lib.kvs_paged_decode_attention(C.byref(c), C.byref(rows(**kw)), None))
    assert "not overlap" in attend(cache(), weights_strides=S2(32, 64)) and "not overlap" in attend(cache(), weights_strides=S2(64, 0))
    assert "must be on device" in attend(cache()) and "must be on device" in attend(cache(), weights=2 * P16, weights_strides=S2(32, 64))
    assert "must be on device" in attend(cache(batch=1), weights_strides=S2(0, 32))
    ev = lambda c, s: error(lib.kvs_evict_paged(C.byref(c), C.byref(_native.EvictRows(
        keep=8, w_len=32, wo_len=32, weights=P16, weights_out=P16, weights_strides=s, weights_out_strides=S2(64, 32))), None))
    assert "not overlap" in ev(cache(), S2(32, 64)) and "must be on device" in ev(cache(batch=1), S2(0, 32))
