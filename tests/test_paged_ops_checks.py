"""Argument checks of the operators on a paged cache that come before any device access (CPU), and
the 64-bit reference of their tests against a plain softmax."""

import ctypes as C

import numpy as np
import pytest
import torch

import paged_ops_reference as R
from kvcache_manager import _native, ops

P16 = 1 << 20  # an aligned address that is never read


def cache(**change):
    c = _native.PagedCache(P16, P16, (C.c_int64 * 3)(4096, 2048, 128), (C.c_int64 * 3)(4096, 2048, 128), P16, 4, 2, 16, 64, 2, 2,
                           _native.DTYPE_BF16, 1.0, 1.0)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def error(rc):
    assert rc == _native.E_INVAL
    return _native.load().kvs_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "cache type 3"), (dict(batch=0), "at least one row"), (dict(batch=65536), "65535"), (dict(block_size=0), "must be > 0"),
    (dict(head_dim=264), "up to 256"), (dict(head_dim=12), "multiple of 8"), (dict(head_dim=24, dtype=2), "multiple of 16"),
    (dict(max_blocks=1 << 28), "2^31"), (dict(num_blocks=1 << 31), "2^31"), (dict(k=P16 + 8), "16-byte"),
    (dict(v_strides=(C.c_int64 * 3)(4096, 2048, 120)), "16-byte"), (dict(k_scale=0.0, dtype=2), "positive and finite"),
    (dict(v_scale=float("nan"), dtype=2), "positive and finite"), (dict(k_scale=2.0), "e4m3 cache"), (dict(page_table=None), "must be on device")])
def test_cache_checks(change, message):
    lib, rows = _native.load(), _native.DecodeRows()
    rows.q_heads = 2
    assert message in error(lib.kvs_paged_decode_attention(C.byref(cache(**change)), C.byref(rows), None))
    assert message in error(lib.kvs_evict_paged(C.byref(cache(**change)), C.byref(_native.EvictRows()), None))
    assert message in error(lib.kvs_qk_norm_rope_fill(C.byref(cache(**change)), C.byref(_native.QkvRows()), None))


def test_rows_checks():
    lib = _native.load()
    assert "null" in error(lib.kvs_paged_decode_attention(C.byref(cache()), None, None))
    assert "null" in error(lib.kvs_paged_decode_attention(None, None, None))
    two = (C.c_int64 * 2)(512, 128)
    d = lambda **kw: C.byref(_native.DecodeRows(**dict(dict(q=P16, out=P16, q_heads=4, dtype=0, scale=1.0, out_strides=two, weights_out_strides=two), **kw)))
    attend = lambda **kw: error(lib.kvs_paged_decode_attention(C.byref(cache()), d(**kw), None))
    assert "same type" in attend(dtype=1) and "bf16 or fp16" in attend(dtype=2) and "multiple of the KV heads" in attend(q_heads=3)
    assert "16-byte" in attend(q=P16 + 2) and "finite" in attend(scale=float("inf")) and "go together" in attend(weights=P16)
    assert "must cover" in attend(weights=P16, weights_out=P16, w_len=31) and "256-byte" in attend(workspace=P16 + 16)
    assert "1024" in attend(q_heads=4096)
    flat = (C.c_int64 * 2)(512, 0)
    assert "broadcast" in attend(out_strides=flat) and "broadcast" in attend(weights=P16, weights_out=P16, w_len=32, weights_out_strides=flat)
    assert "must be on device" in attend()  # host addresses are refused, not read
    f = lambda **kw: C.byref(_native.QkvRows(**dict(dict(q=P16, k=P16, v=P16, q_out=P16, cos_sin=P16, q_heads=4, rotary=64,
                                                         n_positions=8, n_tokens=2, q_out_strides=two), **kw)))
    fill = lambda **kw: error(lib.kvs_qk_norm_rope_fill(C.byref(cache()), f(**kw), None))
    assert "rotary" in fill(rotary=72) and "rotary" in fill(rotary=4) and "at least one row" in fill(n_positions=0)
    assert "eps" in fill(eps=-1.0) and "16-byte" in fill(q_weight=P16 + 4) and "axes" in fill(axes=P16) and "axes" in fill(positions=P16)
    assert "broadcast" in fill(q_out_strides=flat)
    assert "must be on device" in fill()
    assert lib.kvs_qk_norm_rope_fill(C.byref(cache()), f(n_tokens=0), None) == 0
    e = lambda **kw: C.byref(_native.EvictRows(**dict(dict(keep=8, w_len=32, wo_len=32, weights_strides=two, weights_out_strides=two), **kw)))
    evict = lambda **kw: error(lib.kvs_evict_paged(C.byref(cache()), e(**kw), None))
    assert "keep" in evict(keep=0) and "first (5)" in evict(first=5, recent=4) and "must cover keep" in evict(dst_table=P16)
    assert "must cover" in evict(w_len=31) and "must cover" in evict(wo_len=31) and "must be on device" in evict()
    assert "broadcast" in evict(weights_out_strides=flat) and "not overlap" in evict(weights=P16, weights_out=P16, weights_strides=(C.c_int64 * 2)(8, 4))
    single = cache(k_strides=(C.c_int64 * 3)(4096, 0, 128))
    assert "broadcast" in error(lib.kvs_evict_paged(C.byref(single), e(), None)) and "broadcast" in error(lib.kvs_qk_norm_rope_fill(C.byref(single), f(), None))


def test_cpu_tensors_are_refused():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    n = lambda *s: z(*s, dt=torch.int32)
    c = z(4, 2, 16, 64)
    with pytest.raises(RuntimeError, match="must be on device"):
        ops.qk_norm_rope_fill(z(8, 4, 64), z(8, 2, 64), z(8, 2, 64), z(8, 64), n(3), n(2, 2), n(2), c, c)
    with pytest.raises(RuntimeError, match="must be on device"):
        ops.paged_decode_attention(z(2, 4, 64), c, c, n(2, 2), n(2))
    with pytest.raises(RuntimeError, match="must be on device"):
        ops.evict_paged_kv(c, c, n(2, 2), n(2), z(2, 2, 32), 4)


def test_reference_is_the_softmax():
    r = np.random.default_rng(0)
    ck, cv = r.normal(size=(9, 2, 4, 8)), r.normal(size=(9, 2, 4, 8))
    q, table = r.normal(size=(1, 4, 8)), np.array([[3, 0, 8, 5]], np.int32)
    out, lse, w, *_ = R.attend(q, ck, cv, table, [14], 0.5)
    toks = [0, 1, 2, 3, 8, 9, 10, 11, 12, 13]
    k = np.stack([ck[table[0, t // 4], 1, t % 4] for t in toks])
    v = np.stack([cv[table[0, t // 4], 1, t % 4] for t in toks])
    p = torch.softmax(torch.tensor(k @ q[0, 3] * 0.5), 0).numpy()
    assert np.allclose(out[0, 3], p @ v) and np.allclose(lse[0, 3], torch.logsumexp(torch.tensor(k @ q[0, 3] * 0.5), 0).item())
    assert np.allclose(w[0].sum(1), 2) and (w[0, :, 4:8] == 0).all() and (w[0, :, 14:] == 0).all()
    kept, new = R.evict(np.array([[[5.0, 1, 1, 2, 9, 9, 9, 9, 1, 0, 0, 3, 0, 0]]]), table[:, :], [14], 5, 1, 2, 4, 9)
    assert kept.tolist() == [[[0, 3, 11, 12, 13]]] and new.tolist() == [5]
    y, _ = R.rows_of(np.ones((1, 4)), None, 0, np.array([[0.0, 0, 1, 1]]), np.zeros(2, int), 4, True)
    assert y.tolist() == [[-1, 1, -1, 1]]
