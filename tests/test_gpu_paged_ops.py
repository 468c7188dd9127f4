"""The operators on a paged cache (kvcache_manager.ops.qk_norm_rope_fill, paged_decode_attention,
evict_paged_kv) against their 64-bit definitions, within bounds derived in paged_ops_reference.py."""

import numpy as np
import pytest
import torch

import paged_ops_reference as R
from kvcache_manager import ops

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x):
    return torch.as_tensor(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def to_cache(t, layout):
    """t [blocks, heads, size, dim] on the GPU; `nhd`: token-major in memory."""
    return t.cuda().contiguous() if layout == "hnd" else t.transpose(1, 2).contiguous().cuda().transpose(1, 2)


def nans_like(shape, dtype):
    t = torch.full(shape, float("nan"), dtype=torch.float32)
    t[..., ::3] = float("inf")
    return t.to(dtype) if dtype != E4M3 else torch.full(shape, float("nan")).to(dtype)


def cache_of(g, lens, page, heads, dim, dtype, low=None, holes=(), spare=2):
    """K and V [blocks, heads, page, dim] (CPU) and a table: every slot that no token of a request
    holds, and every page that the table does not name, is infinite or NaN."""
    pages_of = [max(0, -(-n // page)) for n in lens]
    total = sum(pages_of)
    blocks = total + spare + 1
    ids = (torch.randperm(total + spare, generator=g)[:total] + 1).numpy()
    table = np.full((len(lens), max(pages_of + [1]) + 1), -1, np.int32)
    k, v = nans_like((blocks, heads, page, dim), dtype), nans_like((blocks, heads, page, dim), dtype)
    at = 0
    for b, n in enumerate(lens):
        for j in range(pages_of[b]):
            pg = int(ids[at])
            at += 1
            if (b, j) in holes:
                table[b, j] = [0, -1, blocks, 2**31 - 1][j % 4]
                continue
            table[b, j] = pg
            s0 = max(0, (low[b] if low else 0) - j * page)
            s1 = min(page, n - j * page)
            if s1 > s0:
                k[pg, :, s0:s1] = (torch.randn((heads, s1 - s0, dim), generator=g)).to(dtype)
                v[pg, :, s0:s1] = (torch.randn((heads, s1 - s0, dim), generator=g)).to(dtype)
    return k, v, table


def check_attend(seed, lens, *, dtype=BF16, cache="same", dim=128, heads=2, group=4, page=64, layout="hnd", window=0,
                 holes=(), weights=False, q_scale=2.0, scale=None):
    g = gen(seed)
    cdt = E4M3 if cache == "fp8" else dtype
    low = [max(0, n - window) if window else 0 for n in lens]
    k, v, table = cache_of(g, lens, page, heads, dim, cdt, low, holes)
    q = (torch.randn((len(lens), heads * group, dim), generator=g) * q_scale).to(dtype)
    ks, vs = (0.37, 1.9) if cache == "fp8" else (1.0, 1.0)
    scale = dim**-0.5 if scale is None else scale
    out, lse, w, b_out, b_lse, b_w = R.attend(R.f64(q), R.f64(k), R.f64(v), table, lens, scale, window, ks, vs, dtype, cache == "fp8")
    kd, vd = to_cache(k, layout), to_cache(v, layout)
    args = {}
    if weights:
        start = torch.rand((len(lens), heads, table.shape[1] * page + 3), generator=g)
        args = dict(weights=start.cuda(), weights_out=torch.full(start.shape, 7.0, device="cuda"))
    call = lambda **kw: ops.paged_decode_attention(q.cuda(), kd, vd, i32(table), i32(lens), scale=scale,
                                                   window=window or None, k_scale=ks, v_scale=vs, return_lse=True, **kw)
    got, got_lse = call(**args)
    got2, lse2 = call()
    assert torch.equal(got, got2) and torch.equal(got_lse, lse2)  # equal calls give equal bits
    got, got_lse = R.f64(got), R.f64(got_lse)
    assert np.isfinite(got).all()
    bad = np.abs(got - out) > b_out
    assert not bad.any(), (np.abs(got - out)[bad].max(), b_out[bad].min(), np.argwhere(bad)[:4])
    empty = np.isinf(lse)
    assert (got_lse[empty] == -np.inf).all() and (np.abs(got_lse[~empty] - lse[~empty]) <= b_lse[~empty]).all()
    if weights:
        gw = R.f64(args["weights_out"])
        for b, n in enumerate(lens):
            want = R.f64(start)[b, :, :n] + w[b, :, :n]
            assert (np.abs(gw[b, :, :n] - want) <= b_w[b, :, :n] + 2.0**-23 * want).all()
            assert (gw[b, :, n:] == 7.0).all()  # nothing behind a request's tokens is written


LENS = [1, 0, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700]


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_head_dims(dim, dtype):
    check_attend(dim, LENS, dtype=dtype, dim=dim, heads=2, group=4, layout="nhd" if dim % 16 else "hnd")


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 208, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_fp8_cache(dim, dtype):
    check_attend(dim + 1, LENS, dtype=dtype, cache="fp8", dim=dim, heads=2, group=5, page=16, layout="nhd")


@pytest.mark.parametrize("group", [1, 7, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_attention_groups(group, cache):
    check_attend(group, [5, 300, 1000], group=group, heads=3, dim=64, cache=cache, weights=True)


@pytest.mark.parametrize("group,dim", [(16, 128), (16, 256), (12, 256)])
def test_attention_wide_groups_and_heads(group, dim):
    check_attend(group + dim, [40, 600], group=group, heads=1, dim=dim, weights=True)


@pytest.mark.parametrize("page", [1, 7, 16, 24, 48, 128, 1000])
@pytest.mark.parametrize("window", [0, 1, 100, 257])
def test_attention_pages_and_windows(page, window):
    check_attend(page + window, [1, 99, 100, 101, 640], page=page, window=window, dim=64, heads=2, group=2, weights=True)


def test_attention_missing_pages():
    """Pages that hold nothing (0, -1) or are out of range, one request without any page left."""
    holes = {(0, 0), (0, 1), (0, 2), (0, 3), (1, 1), (1, 2), (2, 0), (3, 6), (3, 7)}
    check_attend(5, [61, 200, 17, 128], page=16, holes=holes, dim=64, group=3, weights=True)
    check_attend(6, [61, 200, 17, 128], page=20, holes=holes, dim=64, group=3, weights=True)


@pytest.mark.parametrize("heads,dim,length", [(1, 64, 70001), (2, 128, 20000), (1, 256, 9000)])
def test_attention_one_long_request_is_split_and_joined(heads, dim, length):
    check_attend(length, [length], heads=heads, dim=dim, group=2, weights=True)


@pytest.mark.parametrize("batch", [128, 129, 300])
def test_attention_many_requests(batch):
    r = np.random.default_rng(batch)
    check_attend(batch, [int(x) for x in r.integers(0, 600, batch)], dim=64, heads=1, group=2, page=32, weights=True)


def test_attention_peaked_scores():
    """Scores of +-hundreds: the running maximum moves, most probabilities vanish."""
    check_attend(1, [1000, 40], dim=64, group=4, q_scale=40.0, weights=True)
    check_attend(2, [1000, 40], dim=64, group=4, q_scale=40.0, scale=-0.3, weights=True)
    check_attend(3, [1000, 40], dim=64, group=4, q_scale=4e4, cache="fp8", scale=1e-4)
    check_attend(4, [1000, 40], dim=64, group=4, q_scale=1e-6, cache="fp8", dtype=BF16, scale=1e5)


def test_attention_strides_and_given_output():
    """Queries as a slice of a projection, output into a slice, weights into a wider buffer, in place."""
    g = gen(8)
    lens, heads, group, dim, page = [77, 300], 2, 4, 64, 32
    k, v, table = cache_of(g, lens, page, heads, dim, BF16)
    wide = torch.randn((2, (heads * group + 2 * heads) * dim), generator=g).to(BF16).cuda()
    q = wide[:, : heads * group * dim].unflatten(1, (-1, dim))
    kd, vd = to_cache(k, "hnd"), to_cache(v, "nhd")
    store = torch.zeros((2, heads * group, 2 * dim), dtype=BF16, device="cuda")
    wbuf = torch.zeros((2, heads + 1, 400), device="cuda")
    out = ops.paged_decode_attention(q, kd, vd, i32(table), i32(lens), out=store[..., dim:], weights=wbuf[:, :heads])
    ref = ops.paged_decode_attention(q.contiguous(), kd, to_cache(v, "hnd"), i32(table), i32(lens))
    assert out.data_ptr() == store[..., dim:].data_ptr()
    assert torch.equal(out, ref) and (store[..., :dim] == 0).all()
    assert (wbuf[:, heads] == 0).all()
    assert torch.allclose(wbuf[:, :heads].sum(2), torch.full((2, heads), float(group), device="cuda"), atol=1e-4)


def test_attention_reads_broadcast_heads():
    g = gen(19)
    k, v, table = cache_of(g, [70], 16, 1, 64, BF16)
    q = torch.randn((1, 4, 64), generator=g).to(BF16).cuda()
    one = ops.paged_decode_attention(q, k.cuda(), v.cuda(), i32(table), i32([70]))
    two = ops.paged_decode_attention(q, k.cuda().expand(-1, 2, -1, -1), v.cuda().expand(-1, 2, -1, -1), i32(table), i32([70]))
    assert torch.allclose(one.float(), two.float(), atol=2.0**-7)


def test_attention_nan_and_infinite_values_reach_only_their_row():
    g = gen(9)
    k, v, table = cache_of(g, [50, 50], 16, 2, 64, BF16)
    q = torch.randn((2, 4, 64), generator=g).to(BF16)
    v[table[0, 1], 0, 3, 5] = float("nan")
    out, lse = ops.paged_decode_attention(q.cuda(), k.cuda(), v.cuda(), i32(table), i32([50, 50]), return_lse=True)
    assert out[0, :2, 5].isnan().all() and torch.isfinite(lse).all()
    rest = out.clone()
    rest[0, :2, 5] = 0
    assert torch.isfinite(rest).all()
    k[table[1, 0], 1, 2] = float("nan")
    out, lse = ops.paged_decode_attention(q.cuda(), k.cuda(), v.cuda(), i32(table), i32([50, 50]), return_lse=True)
    assert out[1, 2:].isnan().all() and lse[1, 2:].isnan().all() and torch.isfinite(out[1, :2]).all()


def test_attention_rows_of_lowest_scores():
    """Every score -infinity: nothing is attended to, as in a row whose tokens are all masked."""
    g = gen(10)
    k, v, table = cache_of(g, [20], 16, 1, 64, BF16)
    k[table[0, 0]] = 0
    k[table[0, 1]] = 0
    k[..., 0] = -torch.inf
    q = torch.zeros((1, 2, 64), dtype=BF16)
    q[..., 0] = 1
    w = torch.zeros((1, 1, 48), device="cuda")
    out, lse = ops.paged_decode_attention(q.cuda(), k.cuda(), v.cuda(), i32(table), i32([20]), return_lse=True, weights=w)
    assert (out == 0).all() and (lse == -torch.inf).all() and (w == 0).all()


def test_attention_cache_beyond_32_bit_offsets():
    """Pages more than 4 GiB into the cache."""
    heads, page, dim = 8, 64, 128
    blocks = (5 << 30) // (heads * page * dim * 2)
    ck = torch.empty((blocks, heads, page, dim), dtype=BF16, device="cuda")
    cv = torch.empty_like(ck)
    g = gen(11)
    lens = [100, 130]
    k, v, table = cache_of(g, lens, page, heads, dim, BF16)
    q = torch.randn((2, 16, dim), generator=g).to(BF16).cuda()
    ref = ops.paged_decode_attention(q, k.cuda(), v.cuda(), i32(table), i32(lens))
    far = np.where(table > 0, blocks - table, table)
    for p in table[table > 0]:
        ck[blocks - int(p)], cv[blocks - int(p)] = k[int(p)].cuda(), v[int(p)].cuda()
    assert torch.equal(ref, ops.paged_decode_attention(q, ck, cv, i32(far), i32(lens)))


# ------------------------------------------------------------------ norm, rotation and fill


def check_fill(seed, pieces, *, dtype=BF16, cache="same", dim=128, rotary=None, q_heads=4, heads=2, page=16,
               layout="hnd", norm=True, axes=0, interleaved=False, pad=3, in_place=False, bad_positions=False):
    """pieces: (tokens, start) per request. Every element of q_out and of both caches is checked."""
    g = gen(seed)
    cdt = E4M3 if cache == "fp8" else dtype
    rotary = dim if rotary is None else rotary
    total = sum(c for c, _ in pieces)
    t = total + pad
    qkv = torch.randn((t, (q_heads + 2 * heads) * dim + 8), generator=g).to(dtype)[:, 8:]
    q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([q_heads * dim, heads * dim, heads * dim], dim=1))
    blocks = sum(-(-(c + s) // page) for c, s in pieces) + 2
    ck = (torch.randn((blocks, heads, page, dim), generator=g)).to(cdt)
    cv = (torch.randn((blocks, heads, page, dim), generator=g)).to(cdt)
    ids = (torch.randperm(blocks - 1, generator=g) + 1).tolist()
    width = max(-(-(c + s) // page) for c, s in pieces) + 1
    table = np.full((len(pieces) + 1, width), -1, np.int32)  # one request more than cu_seqlens names
    for b, (c, s) in enumerate(pieces):
        for j in range(-(-(c + s) // page)):
            table[b, j] = ids.pop()
    dropped = 0
    if pieces[0][0] > 2:  # one page holds nothing, one is out of range
        table[0, pieces[0][1] // page] = 0
    if len(pieces) > 1:
        table[1, pieces[1][1] // page] = blocks
    cu = np.concatenate([[0], np.cumsum([c for c, _ in pieces]), [-1]]).astype(np.int32)
    starts = np.array([s for _, s in pieces] + [0], np.int32)
    n_pos = max(c + s for c, s in pieces) + 5
    half = rotary // 2
    ang = np.arange(n_pos)[:, None] * (1e4 ** (-np.arange(half) / half))
    cs = torch.tensor(np.concatenate([np.cos(ang), np.sin(ang)], 1), dtype=torch.float32)
    positions = axis_of = None
    if axes:
        positions = torch.randint(0, n_pos, (axes, t), generator=g).to(torch.int32)
        if bad_positions:
            positions[axes - 1, 1] = n_pos
            positions[0, 2] = -1
        axis_of = torch.randint(0, axes, (half,), generator=g).to(torch.int32)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dtype) for _ in range(2)) if norm else (None, None)
    ks, vs = (0.031, 0.07) if cache == "fp8" else (1.0, 1.0)

    want_q, want_k, want_v = np.zeros((t, q_heads, dim)), R.f64(ck), R.f64(cv)
    tol_q, tol_k, tol_v = np.zeros(want_q.shape), np.zeros(want_k.shape), np.zeros(want_v.shape)
    fp32 = (dim + 24) * 2.0**-24
    table_rows = cs.double().numpy()
    f = lambda x: None if x is None else R.f64(x)
    tok = 0
    for b, (c, s) in enumerate(pieces):
        for i in range(c):
            pos = np.full(half, s + i)
            bad = False
            if axes:
                col = positions[:, tok].numpy()
                bad = bool(((col < 0) | (col >= n_pos)).any())
                pos = col[axis_of.numpy()]
            entry = int(table[b, (s + i) // page])
            dropped += bad or entry >= blocks
            if not bad:
                y, mag = R.rows_of(R.f64(q[tok]), f(wq), 1e-6, table_rows, pos, rotary, interleaved)
                want_q[tok], tol_q[tok] = y, R.HALF_STEP[dtype] * np.abs(y) + 1.01 * fp32 * mag + R.TINY[dtype]
                if 0 < entry < blocks:
                    y, mag = R.rows_of(R.f64(k[tok]), f(wk), 1e-6, table_rows, pos, rotary, interleaved)
                    top = R.E4M3_MAX if cache == "fp8" else np.inf
                    row = (s + i) % page
                    y, mag = np.clip(y / ks, -top, top), mag / ks
                    want_k[entry, :, row] = y
                    tol_k[entry, :, row] = R.HALF_STEP[cdt] * np.abs(y) + 1.1 * fp32 * mag + R.TINY[cdt]
                    y = np.clip(R.f64(v[tok]) / vs, -top, top)
                    want_v[entry, :, row] = y
                    tol_v[entry, :, row] = (R.HALF_STEP[cdt] * 1.001 * np.abs(y) + R.TINY[cdt]) if cache == "fp8" else 0
            tok += 1
    dq = qkv.cuda()
    dq, dk, dv = (x.unflatten(1, (-1, dim)) for x in dq.split([q_heads * dim, heads * dim, heads * dim], dim=1))
    before = dq.clone()
    dck, dcv = to_cache(ck, layout), to_cache(cv, layout)
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = lambda x: None if x is None else x.cuda()
    got, rk, rv = ops.qk_norm_rope_fill(dq, dk, dv, cs.cuda(), i32(cu), i32(table), i32(starts), dck, dcv, q_weight=d(wq),
                                        k_weight=d(wk), positions=d(positions), axes=d(axis_of), interleaved=interleaved,
                                        k_scale=ks, v_scale=vs, q_out=dq if in_place else None, out_of_range=count)
    assert rk is dck and rv is dcv
    if in_place:
        assert got is dq and torch.equal(dq[total:], before[total:])  # rows behind the last sequence
        got = torch.cat([got[:total], torch.zeros_like(got[total:])])
    for name, have, want, tol in (("q", got, want_q, tol_q), ("k", dck, want_k, tol_k), ("v", dcv, want_v, tol_v)):
        bad = ~(np.abs(R.f64(have) - want) <= tol)
        assert not bad.any(), (name, np.argwhere(bad)[:5], np.abs(R.f64(have) - want)[bad].max())
    assert int(count.item()) == dropped


PIECES = [(5, 3), (1, 0), (33, 40), (2, 15)]


@pytest.mark.parametrize("dim,rotary", [(8, 8), (64, 64), (64, 32), (80, 40), (96, 96), (128, 128), (128, 64), (200, 200), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_fill_head_dims(dim, rotary, interleaved):
    check_fill(dim + rotary, PIECES, dim=dim, rotary=rotary, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("norm", [True, False])
def test_fill_types_and_layouts(dtype, cache, layout, norm):
    check_fill(3, PIECES, dtype=dtype, cache=cache, layout=layout, norm=norm, q_heads=6, heads=3, dim=64, page=24)
    check_fill(4, PIECES, dtype=dtype, cache=cache, layout=layout, norm=norm, q_heads=5, heads=1, dim=128, interleaved=True)


@pytest.mark.parametrize("axes", [1, 3, 5])
@pytest.mark.parametrize("interleaved", [False, True])
def test_fill_positions_of_several_axes(axes, interleaved):
    check_fill(axes, PIECES, axes=axes, interleaved=interleaved, dim=96, rotary=64, bad_positions=True)


@pytest.mark.parametrize("requests", [1, 31, 32, 33, 1000, 1100])
def test_fill_many_requests(requests):
    r = np.random.default_rng(requests)
    check_fill(requests, [(1, int(s)) for s in r.integers(0, 20, requests)], dim=32, q_heads=2, heads=1, page=8)


def test_fill_in_place_and_many_heads():
    check_fill(7, PIECES, in_place=True, q_heads=64, heads=8, dim=128, page=64)
    check_fill(8, [(300, 0), (77, 9)], in_place=True, q_heads=7, heads=7, dim=64, page=64, pad=0)


def test_fill_matches_paged_fill():
    """Without norm and with a rotation by zero, K and V land where paged_fill_cache_varlen puts them."""
    g = gen(12)
    heads, dim, page, t = 2, 64, 16, 70
    k, v = (torch.randn((t, heads, dim), generator=g).to(BF16).cuda() for _ in range(2))
    cu, sp = i32([0, 30, 65, -1]), i32([5, 0, 0])
    table = i32([[3, 0, 7, 4], [5, 99, 6, -1], [1, 2, 8, 9]])
    one = torch.cat([torch.ones((64, dim // 2)), torch.zeros((64, dim // 2))], 1).cuda()
    a, b = (torch.randn((12, heads, page, dim), generator=g).to(BF16).cuda() for _ in range(2))
    a2, b2 = a.clone(), b.clone()
    n1, n2 = (torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))
    ops.paged_fill_cache_varlen(k.transpose(0, 1)[None].contiguous(), v.transpose(0, 1)[None].contiguous(), cu, table, sp, a, b, out_of_range=n1)
    ops.qk_norm_rope_fill(k, k, v, one, cu, table, sp, a2, b2, out_of_range=n2)
    assert torch.equal(a, a2) and torch.equal(b, b2) and torch.equal(n1, n2) and int(n1) > 0


def test_fill_saturates_and_keeps_nan():
    q = torch.tensor([[[float("nan"), 1e30, -1e30, float("inf")] + [1.0] * 12]], dtype=BF16, device="cuda")
    ck, cv = (torch.zeros((2, 1, 4, 16), dtype=E4M3, device="cuda") for _ in range(2))
    cs = torch.cat([torch.ones((8, 8)), torch.zeros((8, 8))], 1)[:, [0, 1, 2, 3, 8, 9, 10, 11]].contiguous().cuda()
    ops.qk_norm_rope_fill(q, q, q, cs, i32([0, 1]), i32([[1]]), i32([2]), ck, cv)
    row = cv[1, 0, 2].float()
    assert row[0].isnan() and row[1:4].tolist() == [448.0, -448.0, 448.0] and (row[4:] == 1).all()


def test_fill_no_tokens():
    z = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    c = torch.ones((2, 2, 16, 64), dtype=BF16, device="cuda")
    q, _, _ = ops.qk_norm_rope_fill(z, z, z, torch.zeros((4, 64), device="cuda"), i32([0, 0]), i32([[1]]), i32([0]), c, c.clone())
    assert q.shape == (0, 2, 64) and (c == 1).all()


# ------------------------------------------------------------------ eviction


def check_evict(seed, lens, keep, *, first=0, recent=0, heads=2, dim=64, page=16, layout="hnd", dtype=BF16, in_place=False,
                holes=(), ties=True, extra=5):
    g = gen(seed)
    k, v, table = cache_of(g, lens, page, heads, dim, dtype, holes=holes, spare=2 + sum(-(-min(n, keep) // page) for n in lens))
    blocks = k.shape[0]
    cover = table.shape[1] * page
    w = torch.rand((len(lens), heads, cover + extra), generator=g)
    if ties:
        w = (w * 8).floor() / 4 - 0.5
        w[torch.rand(w.shape, generator=g) < 0.05] = -0.0
    w[torch.rand(w.shape, generator=g) < 0.01] = float("inf")
    w[torch.rand(w.shape, generator=g) < 0.01] = float("nan")
    w[torch.rand(w.shape, generator=g) < 0.01] = -float("inf")
    want, new = R.evict(w.double().numpy(), table, lens, keep, first, recent, page, blocks)
    free = [p for p in range(1, blocks) if p not in set(table.ravel().tolist())]
    width = -(-min(keep, cover) // page)
    dst = table if in_place else np.full((len(lens), width), -1, np.int32)
    if not in_place:
        for b, n in enumerate(lens):
            for j in range(-(-min(n, keep) // page)):
                dst[b, j] = free.pop()
    bits = lambda t: t.contiguous().view(torch.uint8).cpu().numpy()
    wk, wv, ww = bits(k).copy(), bits(v).copy(), w.numpy().copy()
    sk, sv = bits(k), bits(v)
    lost = 0
    for b, n in enumerate(lens):
        for h in range(heads):
            m = int(new[b])
            ww[b, h, :m] = w[b, h, want[b, h, :m]].numpy()
            ww[b, h, m:max(0, min(n, cover))] = 0
            for i in range(m):
                t = int(want[b, h, i])
                sp, dp = R.token_page(table, b, t, page, blocks), R.token_page(dst, b, i, page, blocks)
                if dp is None:
                    lost += h == 0
                    continue
                wk[dp, h, i % page], wv[dp, h, i % page] = sk[sp, h, t % page], sv[sp, h, t % page]
    kd, vd, wd = to_cache(k, layout), to_cache(v, layout), w.cuda()
    w_out = wd if in_place else wd.clone()
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    kept, lens_out = ops.evict_paged_kv(kd, vd, i32(table), i32(lens), wd, keep, first=first, recent=recent,
                                        dst_page_table=None if in_place else i32(dst), weights_out=None if in_place else w_out,
                                        out_of_range=count)
    assert np.array_equal(lens_out.cpu().numpy(), new)
    assert np.array_equal(kept.cpu().numpy(), want)
    assert np.array_equal(w_out.cpu().numpy().view(np.uint32), ww.view(np.uint32))
    assert np.array_equal(bits(kd), wk) and np.array_equal(bits(vd), wv)
    assert int(count.item()) == lost


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 1, 0), (16, 2, 5), (64, 0, 64), (100, 4, 30), (2000, 4, 8)])
def test_evict(keep, first, recent, in_place):
    check_evict(keep, [0, 1, 17, 64, 100, 333, 1200], keep, first=first, recent=recent, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dim,page,layout,dtype", [(8, 7, "nhd", BF16), (80, 48, "hnd", FP16), (256, 64, "nhd", BF16), (48, 16, "nhd", E4M3)])
def test_evict_layouts(dim, page, layout, dtype, in_place):
    check_evict(dim, [90, 5, 260], 60, first=3, recent=7, dim=dim, page=page, layout=layout, dtype=dtype, in_place=in_place, heads=3)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,keep", [([3, 4, 5, 97], 4), ([900, 2050, 0, 1023], 300), ([6001], 2500)])
def test_evict_weights_on_16_byte_rows(lens, keep, in_place):
    check_evict(keep, lens, keep, first=1, recent=2, in_place=in_place, page=16, dim=16, extra=0)
    check_evict(keep, lens, keep, first=1, recent=2, in_place=in_place, page=18, dim=16, extra=(-(max(lens) // 18 + 2) * 18) % 4, ties=False)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_missing_pages(in_place):
    holes = {(0, 0), (0, 1), (0, 2), (1, 1), (1, 3), (2, 0)}
    check_evict(21, [45, 100, 90, 50], 30, first=5, recent=10, holes=holes, in_place=in_place)
    check_evict(22, [45, 100, 90, 50], 200, first=5, recent=10, holes=holes, in_place=in_place)


@pytest.mark.parametrize("length,keep", [(9000, 4000), (20000, 777), (66000, 30000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_long_rows(length, keep, in_place):
    check_evict(length, [length, length // 3], keep, first=4, recent=100, heads=1, dim=16, page=64, in_place=in_place, ties=length == 9000)


def test_evict_row_longer_than_a_cluster_holds():
    """More tokens than 8 CTAs keep in shared memory: the weights are read again by each pass."""
    n, page = 8 * 49152 + 1000, 4096
    g = gen(31)
    w = torch.rand((1, 1, page * 98), generator=g).cuda()
    table = i32(np.concatenate([np.arange(1, 99)])[None])
    ck, cv = (torch.zeros((100, 1, page, 8), dtype=BF16, device="cuda") for _ in range(2))
    old = w.clone()
    kept, lens = ops.evict_paged_kv(ck, cv, table, i32([n]), w, 1000, first=2, recent=3, dst_page_table=i32([[99]]))
    after, w = w, old
    other = torch.full_like(w, 5)
    again, _ = ops.evict_paged_kv(ck, cv, table, i32([n]), w, 1000, first=2, recent=3, dst_page_table=i32([[99]]), weights_out=other)
    key = w[0, 0, :n].clone()
    key[:2] = 9
    key[-3:] = 9
    want = torch.sort(torch.sort(key, descending=True, stable=True).indices[:1000]).values
    assert int(lens[0]) == 1000 and torch.equal(kept[0, 0].long(), want) and torch.equal(again, kept)
    assert torch.equal(after[0, 0, :1000], w[0, 0, want]) and (after[0, 0, 1000:n] == 0).all() and torch.equal(after[0, 0, n:], w[0, 0, n:])
    assert torch.equal(other[0, 0, :n], after[0, 0, :n]) and (other[0, 0, n:] == 5).all()


# ------------------------------------------------------------------ a run of them, streams, graphs


def test_decode_loop_against_64_bits():
    """Prefill, decode steps that collect weights, eviction to fresh pages, further steps with the
    tokens' own positions: what a user runs, against 64 bits on the caches that the kernels wrote."""
    g = gen(40)
    heads, group, dim, page, batch, keep = 2, 4, 64, 16, 3, 40
    hq, blocks = heads * group, 80
    ck, cv = (nans_like((blocks, heads, page, dim), BF16).cuda() for _ in range(2))
    ids = (torch.randperm(blocks - 1, generator=g) + 1).tolist()
    table = np.full((batch, 8), -1, np.int32)
    for b in range(batch):
        table[b, :6] = [ids.pop() for _ in range(6)]
    half = dim // 2
    ang = np.arange(256)[:, None] * (1e4 ** (-np.arange(half) / half))
    cs = torch.tensor(np.concatenate([np.cos(ang), np.sin(ang)], 1), dtype=torch.float32).cuda()
    wq, wk = ((1 + 0.1 * torch.randn(dim, generator=g)).to(BF16).cuda() for _ in range(2))
    weights = torch.zeros((batch, heads, 8 * page), device="cuda")
    lens = np.array([50, 7, 81], np.int32)

    def rows(n):
        return [torch.randn((n, h, dim), generator=g).to(BF16).cuda() for h in (hq, heads, heads)]

    q, k, v = rows(int(lens.sum()))
    cu = np.concatenate([[0], np.cumsum(lens)])
    ops.qk_norm_rope_fill(q, k, v, cs, i32(cu), i32(table), i32([0] * batch), ck, cv, q_weight=wq, k_weight=wk)
    position = lens.copy()
    total = np.zeros((batch, heads, 8 * page))
    for step in range(6):
        q, k, v = rows(batch)
        q, _, _ = ops.qk_norm_rope_fill(q, k, v, cs, i32(range(batch + 1)), i32(table), i32(lens), ck, cv, q_weight=wq,
                                        k_weight=wk, positions=i32(position))
        lens, position = lens + 1, position + 1
        out, lse = ops.paged_decode_attention(q, ck, cv, i32(table), i32(lens), return_lse=True, weights=weights)
        want, want_lse, w, b_out, b_lse, b_w = R.attend(R.f64(q), R.f64(ck), R.f64(cv), table, lens, dim**-0.5)
        assert (np.abs(R.f64(out) - want) <= b_out).all() and (np.abs(R.f64(lse) - want_lse) <= b_lse).all()
        total += w
        assert np.allclose(R.f64(weights), total, rtol=2.0**-20, atol=float(b_w.max()) * 8)
        if step == 2:
            fresh = np.full((batch, 8), -1, np.int32)
            for b in range(batch):
                fresh[b, :4] = [ids.pop() for _ in range(4)]
            kept, new = R.evict(R.f64(weights), table, lens, keep, 4, 8, page, blocks)
            got, got_lens = ops.evict_paged_kv(ck, cv, i32(table), i32(lens), weights, keep, first=4, recent=8, dst_page_table=i32(fresh))
            assert np.array_equal(got.cpu().numpy(), kept) and np.array_equal(got_lens.cpu().numpy(), new)
            for b in range(batch):
                for h in range(heads):
                    total[b, h, : new[b]] = total[b, h, kept[b, h, : new[b]]]
                    total[b, h, new[b]:] = 0
            table, lens = fresh, new.copy()


def small_case(seed):
    g = gen(seed)
    lens = [300, 40, 0, 777]
    k, v, table = cache_of(g, lens, 16, 2, 64, BF16, spare=60)
    q = torch.randn((4, 8, 64), generator=g).to(BF16).cuda()
    w = torch.rand((4, 2, table.shape[1] * 16), generator=g).cuda()
    free = sorted(set(range(1, k.shape[0])) - set(table.ravel().tolist()))
    dst = np.full((4, 7), -1, np.int32)
    for b, n in enumerate(lens):
        for j in range(-(-min(n, 100) // 16)):
            dst[b, j] = free.pop()
    return dict(q=q, k=k.cuda(), v=v.cuda(), table=i32(table), lens=i32(lens), w=w, dst=i32(dst))


def attend_and_evict(s, w_out, w_new):
    out, lse = ops.paged_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], return_lse=True, weights=s["w"], weights_out=w_out)
    kept, lens = ops.evict_paged_kv(s["k"], s["v"], s["table"], s["lens"], w_out, 100, first=2, recent=9,
                                    dst_page_table=s["dst"], weights_out=w_new)
    return out, lse, kept, lens


def test_two_captured_graphs_and_an_eager_call():
    """Two graphs captured on one pool, replayed in turn with eager calls between, on changed inputs."""
    cases = [small_case(50), small_case(51)]
    buf = [(torch.zeros_like(s["w"]), torch.zeros_like(s["w"])) for s in cases]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for s, (a, b) in zip(cases, buf):
            attend_and_evict(s, a, b)
    torch.cuda.synchronize()
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for s, (a, b) in zip(cases, buf):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(attend_and_evict(s, a, b))
        graphs.append(graph)
    for round_ in range(3):
        for i in (0, 1):
            s = cases[i]
            s["q"].copy_(torch.randn(s["q"].shape, generator=gen(60 + round_)).to(BF16))
            s["lens"].copy_(i32([[300, 40, 0, 777], [1, 0, 33, 500], [299, 39, 0, 20]][round_]))
            graphs[i].replay()
            got = [x.clone() for x in outs[i]] + [x.clone() for x in buf[i]]
            a, b = torch.zeros_like(s["w"]), torch.zeros_like(s["w"])
            a.copy_(buf[i][0])  # rows behind a request's tokens stay as they were
            b.copy_(buf[i][1])
            want = [*attend_and_evict(s, a, b), a, b]
            for x, y in zip(got, want):
                assert torch.equal(x, y)


def test_calls_on_two_streams_at_once():
    cases = [small_case(70 + i) for i in range(4)]
    ref = []
    for s in cases:
        a, b = torch.zeros_like(s["w"]), torch.zeros_like(s["w"])
        ref.append([*attend_and_evict(s, a, b), a, b])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None] * 4
    for _ in range(20):
        for i, (s, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                a, b = torch.zeros_like(s["w"]), torch.zeros_like(s["w"])
                got[i] = [*attend_and_evict(s, a, b), a, b]
    torch.cuda.synchronize()
    for x, y in zip(ref, got):
        assert all(torch.equal(p, r) for p, r in zip(x, y))


def test_refusals():
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")
    n = lambda *s: z(*s, dt=torch.int32)
    fill = dict(q=z(8, 4, 64), k=z(8, 2, 64), v=z(8, 2, 64), cos_sin=z(16, 64, dt=torch.float32), cu_seqlens=n(3),
                page_table=n(2, 2), start_positions=n(2), cache_k=z(4, 2, 16, 64), cache_v=z(4, 2, 16, 64))
    ops.qk_norm_rope_fill(**fill)
    for change, msg in [(dict(q=z(8, 4, 64).cpu()), "q must be on device"), (dict(k=z(7, 2, 64)), "q's tokens"),
                        (dict(k=z(8, 3, 64), v=z(8, 3, 64)), "cache's heads"), (dict(q=z(8, 4, 32)), "head_dim"),
                        (dict(q=z(8, 4, 64, dt=FP16)), "same dtype"), (dict(cos_sin=z(16, 64)), "float32"),
                        (dict(cos_sin=z(16, 72, dt=torch.float32)), "rotary"), (dict(cos_sin=z(16, 12, dt=torch.float32)), "rotary"),
                        (dict(cos_sin=z(0, 64, dt=torch.float32)), "at least one row"),
                        (dict(cu_seqlens=n(2)), "batch_size \\+ 1"), (dict(start_positions=n(3)), "must match batch_size"),
                        (dict(page_table=z(2, 2)), "INT32"), (dict(page_table=n(0, 2), start_positions=n(0), cu_seqlens=n(1)), "at least one row"),
                        (dict(cache_v=z(4, 2, 16, 64, dt=FP16)), "same shape and dtype"),
                        (dict(cache_k=z(4, 2, 16, 64, dt=FP16), cache_v=z(4, 2, 16, 64, dt=FP16)), "same type"),
                        (dict(cache_k=z(4, 2, 16, 64, dt=torch.float32), cache_v=z(4, 2, 16, 64, dt=torch.float32)), "must be bfloat16"),
                        (dict(cache_k=z(4, 2, 16, 128)[..., ::2], cache_v=z(4, 2, 16, 128)[..., ::2]), "rows must be contiguous"),
                        (dict(cache_k=z(4, 2, 16, 66)[..., 2:], cache_v=z(4, 2, 16, 66)[..., 2:]), "16-byte"),
                        (dict(q=z(8, 4, 66)[..., 2:]), "16-byte"), (dict(k_scale=2.0), "e4m3"), (dict(q_weight=z(32)), "q_weight"),
                        (dict(positions=n(2, 8)), "need axes"), (dict(positions=n(7)), "positions must be"),
                        (dict(positions=n(2, 8), axes=n(31)), "rotary / 2"), (dict(axes=n(32)), "only with positions"),
                        (dict(positions=n(33, 8), axes=n(32)), "32 axes"), (dict(eps=-1.0), "eps"), (dict(q_out=z(8, 4, 32)), "q_out"),
                        (dict(out_of_range=z(1)), "int32"), (dict(q_out=z(1, 4, 64).expand(8, 4, 64)), "broadcast"),
                        (dict(cache_v=z(1, 2, 16, 64).expand(4, 2, 16, 64)), "broadcast"), (dict(q=z(8, 4, 64).requires_grad_()), "no backward")]:
        with pytest.raises(RuntimeError, match=msg):
            ops.qk_norm_rope_fill(**dict(fill, **change))
    att = dict(q=z(2, 4, 64), cache_k=z(4, 2, 16, 64), cache_v=z(4, 2, 16, 64), page_table=n(2, 2), seq_lens=n(2))
    ops.paged_decode_attention(**att)
    f32 = lambda *s: z(*s, dt=torch.float32)
    for change, msg in [(dict(q=z(3, 4, 64)), "requests"), (dict(q=z(2, 3, 64)), "multiple of the KV heads"), (dict(seq_lens=n(3)), "must match"),
                        (dict(seq_lens=f32(2)), "INT32"), (dict(window=0), "window"), (dict(scale=float("nan")), "scale"),
                        (dict(out=z(2, 4, 32)), "out must"), (dict(out=z(2, 1, 64).expand(2, 4, 64)), "broadcast"),
                        (dict(weights=f32(2, 1, 32).expand(2, 2, 32)), "broadcast"), (dict(weights=f32(2, 2, 31)), "must cover"), (dict(weights=f32(2, 4, 32)), "num_kv_heads"),
                        (dict(weights_out=f32(2, 2, 32)), "needs weights"), (dict(q=z(2, 4, 64, dt=torch.float32)), "rows must be"),
                        (dict(cache_k=z(4, 2, 16, 512), cache_v=z(4, 2, 16, 512), q=z(2, 4, 512)), "up to 256"),
                        (dict(cache_k=z(4, 2, 16, 24, dt=E4M3), cache_v=z(4, 2, 16, 24, dt=E4M3), q=z(2, 4, 24)), "multiple of 16"),
                        (dict(page_table=n(2, 1 << 28)), "2\\^31")]:
        with pytest.raises(RuntimeError, match=msg):
            ops.paged_decode_attention(**dict(att, **change))
    ev = dict(cache_k=z(4, 2, 16, 64), cache_v=z(4, 2, 16, 64), page_table=n(2, 2), seq_lens=n(2), weights=f32(2, 2, 32), keep=8)
    ops.evict_paged_kv(**ev)
    for change, msg in [(dict(keep=0), "keep"), (dict(first=5, recent=4), "first"), (dict(recent=-1), "recent"), (dict(weights=f32(2, 2, 30)), "must cover"),
                        (dict(dst_page_table=n(1, 1)), "batch_size"), (dict(dst_page_table=n(2, 1), keep=17), "must cover keep"),
                        (dict(weights_out=f32(2, 2, 16)), "must cover"), (dict(cache_k=z(4, 1, 16, 64).expand(4, 2, 16, 64)), "broadcast"),
                        (dict(seq_lens=n(1)), "must match")]:
        with pytest.raises(RuntimeError, match=msg):
            ops.evict_paged_kv(**dict(ev, **change))


def run_all_three(s):
    """Every operator once, with every argument given, on copies of the case's buffers."""
    k, v, w = s["k"].clone(), s["v"].clone(), s["w"].clone()
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = gen(3)
    q, kk, vv = (torch.randn((4, h, 64), generator=g).to(BF16).cuda() for h in (8, 2, 2))
    ones = torch.ones(64, dtype=BF16, device="cuda")
    cs = torch.rand((16, 64), generator=g).cuda()
    out = torch.zeros_like(q)
    new, _, _ = ops.qk_norm_rope_fill(q, kk, vv, cs, i32(range(5)), s["table"], i32([299, 39, 0, 776]), k, v, q_weight=ones,
                                      k_weight=ones, eps=1e-5, positions=i32([[1, 2, 3, 4], [5, 6, 7, 99]]), axes=i32([0, 1] * 16),
                                      interleaved=True, q_out=out, out_of_range=count)
    assert new is out
    att, lse = ops.paged_decode_attention(new, k, v, s["table"], s["lens"], scale=0.3, window=500, out=torch.zeros_like(q), return_lse=True, weights=w)
    plain = ops.paged_decode_attention(new, k, v, s["table"], s["lens"])
    kept, lens = ops.evict_paged_kv(k, v, s["table"], s["lens"], w, 100, first=1, recent=2, dst_page_table=s["dst"], out_of_range=count)
    placed, _ = ops.evict_paged_kv(k, v, s["dst"], lens, w[..., :112].clone(), 50)
    return [new, att, lse, plain, kept, lens, placed, w, count, k.nan_to_num(), v.nan_to_num()]


def test_compiled_and_ctypes_calls_agree(monkeypatch):
    from kvcache_manager import _native

    s = small_case(90)
    assert _native.load_opcall(), "the compiled entry is built beside the library"
    with monkeypatch.context() as m:
        m.setattr(ops, "_paged_cache", None)  # the ctypes path cannot be taken
        fast = run_all_three(s)
    with monkeypatch.context() as m:
        m.setattr(_native, "opcall", False)
        slow = run_all_three(s)
    assert all(torch.equal(a, b) for a, b in zip(fast, slow)) and int(fast[8]) == 1
