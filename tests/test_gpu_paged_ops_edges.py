"""The operators on a paged cache at their edges: probabilities far below a row's largest, errors of a
launch, tensors that autograd watches, and tables and sums that alias. 64-bit definitions and bounds are
those of paged_ops_reference.py."""

import ctypes as C

import numpy as np
import pytest
import torch

import paged_ops_reference as R
from kvcache_manager import _native, ops

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x):
    return torch.as_tensor(np.ascontiguousarray(x, dtype=np.int32)).cuda()


@pytest.mark.parametrize("nats", [11, 15, 17, 19])
@pytest.mark.parametrize("dtype,fp8", [(FP16, False), (FP16, True), (BF16, True)])
@pytest.mark.parametrize("batch,length", [(40, 512), (1, 4096)])
def test_attention_behind_a_sink(batch, length, dtype, fp8, nats):
    """The first token's score is `nats` above the others' and its value is zero, so that the others'
    probabilities, of e^-nats each, make up the whole output. The 512-token rows are a CTA each, 128 tokens
    sharing the sink's warp; the long row is split."""
    g, page, dim, group = gen(nats), 16, 64, 2
    pages = length // page
    table = (torch.randperm(batch * pages, generator=g) + 1).reshape(batch, pages).numpy().astype(np.int32)
    shape = (batch * pages + 1, 1, page, dim)
    k = 0.05 * torch.randn(shape, generator=g)
    v = (300 + 50 * torch.randn(shape, generator=g)).clamp(150, 440)
    k[table[:, 0], 0, 0] = nats * dim**-0.5
    v[table[:, 0], 0, 0] = 0
    q = (1 + 0.1 * torch.randn((batch, group, dim), generator=g)).to(dtype)
    ks, vs = (0.0625, 1.0) if fp8 else (1.0, 1.0)
    k, v = ((k / ks).to(E4M3), v.to(E4M3)) if fp8 else (k.to(dtype), v.to(dtype))
    lens = [length] * batch
    out, _, _, b_out, _, _ = R.attend(R.f64(q), R.f64(k), R.f64(v), table, lens, dim**-0.5, 0, ks, vs, dtype, fp8)
    # The bound allows each fp16 probability half of the smallest fp16 step, 2^-25, relative to the largest
    # one. Held 2^15 times larger (at most 2^15 < 65504), it is off by half a step of itself, which the bound
    # holds already, or by 2^-25 2^-15 of the largest.
    top = np.abs(R.f64(v)).max() * vs
    b_out = b_out - length * 2.0**-25 * top + length * 2.0**-40 * top
    assert (b_out < 0.05 * np.abs(out)).all()  # what the bound leaves is small beside the output
    got = R.f64(ops.paged_decode_attention(q.cuda(), k.cuda(), v.cuda(), i32(table), i32(lens), k_scale=ks, v_scale=vs))
    assert (np.abs(got - out) <= b_out).all(), (np.abs(got - out) / np.abs(out)).max()


def decode_args(q_heads=4, dim=64):
    """Arguments of the three operators on one small cache (2 requests, 2 KV heads, pages of 16)."""
    g = gen(1)
    randn = lambda *s: torch.randn(s, generator=g).to(BF16).cuda()
    ck, cv = randn(8, 2, 16, dim), randn(8, 2, 16, dim)
    table = i32([[1, 2], [3, 4]])
    angle = torch.rand((64, dim // 2), generator=g)
    fill = dict(q=randn(2, q_heads, dim), k=randn(2, 2, dim), v=randn(2, 2, dim),
                cos_sin=torch.cat([angle.cos(), angle.sin()], 1).cuda(), cu_seqlens=i32([0, 1, 2]), page_table=table,
                start_positions=i32([28, 17]), cache_k=ck, cache_v=cv)
    attend = dict(q=randn(2, q_heads, dim), cache_k=ck, cache_v=cv, page_table=table, seq_lens=i32([29, 18]),
                  weights=torch.rand((2, 2, 32), generator=g).cuda())
    evict = dict(cache_k=ck, cache_v=cv, page_table=table, seq_lens=i32([29, 18]), weights=torch.rand((2, 2, 32), generator=g).cuda(),
                 keep=10, dst_page_table=i32([[5], [6]]))
    return fill, attend, evict


@pytest.mark.parametrize("which", ["fill", "attend", "evict"])
def test_failed_launch_is_reported_and_not_repeated(which, monkeypatch):
    """An error that is no refusal of the arguments ends the call: part of its work may have been
    enqueued. Entry points that only return such an error stand in for the library's."""
    opcall = _native.load_opcall()
    assert opcall
    lib, calls = _native.load(), []
    args = dict(zip(("fill", "attend", "evict"), decode_args()))[which]
    operator = {"fill": ops.qk_norm_rope_fill, "attend": ops.paged_decode_attention, "evict": ops.evict_paged_kv}[which]
    addr = lambda fn: C.cast(fn, C.c_void_p).value
    real = [addr(f) for f in (lib.kvs_qk_norm_rope_fill, lib.kvs_decode_attention_workspace, lib.kvs_paged_decode_attention, lib.kvs_evict_paged)]

    @C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_void_p, C.c_void_p)
    def failing(cache, rows, stream):
        calls.append("compiled")
        return _native.E_CUDA

    class Repeats:  # what the ctypes path would call
        def __getattr__(self, name):
            if name in ("kvs_qk_norm_rope_fill", "kvs_paged_decode_attention", "kvs_evict_paged"):
                return lambda *a: calls.append("repeated") or _native.OK
            return getattr(lib, name)

    monkeypatch.setattr(ops, "load", lambda: Repeats())
    opcall.bind(addr(failing), real[1], addr(failing), addr(failing))
    try:
        with pytest.raises(_native.KvsError) as e:
            operator(**args)
    finally:
        opcall.bind(*real)
    assert calls == ["compiled"] and e.value.code == _native.E_CUDA


@pytest.mark.parametrize("compiled", [True, False])
def test_error_of_an_earlier_call_is_not_taken_for_the_launches(compiled, monkeypatch):
    """A call that failed and said so (a device that is not there) leaves nothing behind: the next ones
    run once and report success."""
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    lib = _native.load()

    def earlier_failure():
        cache = _native.PagedCache(1 << 20, 1 << 20, (C.c_int64 * 3)(4096, 2048, 128), (C.c_int64 * 3)(4096, 2048, 128), 1 << 20, 4, 2, 16, 64,
                                   2, 2, _native.DTYPE_BF16, 1.0, 1.0)
        rows = _native.DecodeRows(q_heads=4)
        assert lib.kvs_decode_attention_workspace(C.byref(cache), C.byref(rows), 999, C.byref(C.c_uint64())) == _native.E_CUDA

    fill, attend, _ = decode_args()
    want, _, _ = ops.qk_norm_rope_fill(**fill)
    out = ops.paged_decode_attention(**dict(attend, weights=None))
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    fill["page_table"] = i32([[1, 99], [3, 4]])  # a token in a page that is not there is counted once
    earlier_failure()
    got, _, _ = ops.qk_norm_rope_fill(**fill, q_out=fill["q"], out_of_range=count)  # in place: turned once
    assert torch.equal(got, want) and int(count) == 1
    earlier_failure()
    assert torch.equal(ops.paged_decode_attention(**dict(attend, weights=None)), out)


def test_failed_server_leaves_no_error_behind():
    """A server whose slab no GPU holds is refused; the next launch of the library is not blamed for it."""
    lib = _native.load()
    config = _native.ServerConfig()
    assert lib.kvs_server_config_default(C.byref(config)) == _native.OK
    config.heap_bytes, config.unit_bytes, config.max_keys, config.host_pool_bytes = 1 << 46, 1 << 24, 64, 0
    server = C.c_void_p()
    assert lib.kvs_server_create(C.byref(config), C.byref(server)) == _native.E_NOSPACE
    k = torch.ones((1, 2, 4, 64), dtype=BF16, device="cuda")
    ck, cv = (torch.zeros((3, 2, 16, 64), dtype=BF16, device="cuda") for _ in range(2))
    ops.paged_fill_cache_varlen(k, k, i32([0, 4]), i32([[2]]), i32([3]), ck, cv)
    assert (ck[2, :, 3:7] == 1).all() and ck.sum() == 2 * 4 * 64


@pytest.mark.parametrize("compiled", [True, False])
def test_tangents_are_refused(compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    fill, attend, evict = decode_args()
    for operator, args, names in ((ops.qk_norm_rope_fill, fill, ("q", "k", "v", "cos_sin", "cache_k")),
                                  (ops.paged_decode_attention, attend, ("q", "cache_v", "weights")), (ops.evict_paged_kv, evict, ("weights",))):
        for name in names:
            with torch.autograd.forward_ad.dual_level():
                dual = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
                with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
                    operator(**dict(args, **{name: dual}))
        operator(**args)


@pytest.mark.parametrize("compiled", [True, False])
def test_written_tensors_count_as_changed(compiled, monkeypatch):
    """autograd refuses a backward pass through a tensor that a call has overwritten since."""
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    fill, attend, evict = decode_args()
    count = lambda: torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(attend["q"])
    sums = torch.zeros_like(attend["weights"])
    calls = [(ops.qk_norm_rope_fill, dict(fill, q_out=fill["q"], out_of_range=count()), ("q", "cache_k", "cache_v", "out_of_range"), ("k", "cos_sin")),
             (ops.paged_decode_attention, dict(attend, out=out), ("out", "weights"), ("q", "cache_k", "cache_v")),
             (ops.paged_decode_attention, dict(attend, weights_out=sums), ("weights_out",), ("weights",)),
             (ops.evict_paged_kv, dict(evict, out_of_range=count()), ("cache_k", "cache_v", "weights", "out_of_range"), ("seq_lens", "dst_page_table")),
             (ops.evict_paged_kv, dict(evict, weights_out=sums), ("weights_out",), ("weights",))]
    for operator, args, written, kept in calls:
        before = {name: args[name]._version for name in written + kept}
        operator(**args)
        assert all(args[name]._version > before[name] for name in written), (operator, written)
        assert all(args[name]._version == before[name] for name in kept), (operator, kept)
    x = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    fill, _, _ = decode_args()
    y = (fill["q"] * x).sum()
    ops.qk_norm_rope_fill(**fill, q_out=fill["q"])
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()


@pytest.mark.parametrize("compiled", [True, False])
def test_inference_tensors_are_written(compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    with torch.inference_mode():
        fill, attend, evict = decode_args()
    want, _, _ = ops.qk_norm_rope_fill(**fill)
    with torch.inference_mode():
        for operator, args in ((ops.paged_decode_attention, attend), (ops.evict_paged_kv, evict)):
            operator(**args)
    got, _, _ = ops.qk_norm_rope_fill(**fill, q_out=fill["q"])
    assert torch.equal(got, want)


@pytest.mark.parametrize("compiled", [True, False])
def test_evict_destination_that_is_the_front_of_the_table(compiled, monkeypatch):
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    g = gen(5)
    ck, cv = (torch.randn((10, 2, 16, 64), generator=g).to(BF16).cuda() for _ in range(2))
    w = torch.rand((1, 2, 128), generator=g).cuda()
    table, lens = i32([[4, 2, 9, 1, 7, 3, 5, 8]]), i32([120])
    call = lambda dst, keep=40: [x for c in ([ck.clone(), cv.clone(), w.clone()],)
                                 for x in (*ops.evict_paged_kv(c[0], c[1], table, lens, c[2], keep, recent=8, dst_page_table=dst), *c)]
    with pytest.raises(RuntimeError, match="must cover keep"):
        call(table[:, :2])
    want = call(None)
    for dst in (table, table[:, :3]):
        assert all(torch.equal(a, b) for a, b in zip(call(dst), want))


@pytest.mark.parametrize("compiled", [True, False])
def test_evict_destination_without_columns(compiled, monkeypatch):
    """A given table that holds no slots is refused; it does not mean in place."""
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    _, _, evict = decode_args()
    before = evict["cache_k"].clone()
    with pytest.raises(RuntimeError, match="must cover keep"):
        ops.evict_paged_kv(**dict(evict, dst_page_table=torch.empty((2, 0), dtype=torch.int32, device="cuda")))
    assert torch.equal(evict["cache_k"], before)


@pytest.mark.parametrize("compiled", [True, False])
def test_fill_positions_without_axes_of_any(compiled, monkeypatch):
    """Given positions of no axis are refused; they do not mean the cache's positions."""
    if not compiled:
        monkeypatch.setattr(_native, "opcall", False)
    fill, _, _ = decode_args()
    before = fill["cache_k"].clone()
    with pytest.raises(RuntimeError, match="positions must be"):
        ops.qk_norm_rope_fill(**fill, positions=torch.empty((0, 2), dtype=torch.int32, device="cuda"))
    assert torch.equal(fill["cache_k"], before)
