"""Chunk gather / scatter ops over paged KV members, the token-granular paged fill, and what a
serving step computes on the paged caches: norm, rotation and fill of new tokens
(`qk_norm_rope_fill`), attention of one new token per request (`paged_decode_attention`) and eviction
by accumulated attention weight (`evict_paged_kv`). All take torch CUDA tensors.

B200 counterparts of ttnn.kvcache_manager.gather_tp_shards_to_chip / scatter_chunk_from_chip /
pack_local_shards / unpack_local_shards (patch 0003 gather.hpp lines 9335-9453). A "rank" is a
GPU that owns one TP shard of every member; `members[r][m]` is rank r's shard of member m. The
master GPU (the device of `dst` / `src`) moves every byte with one kernel, reading or writing the
other ranks' shards over NVLink peer access. Layout: for member m, chunk block cb and rank r, the
shard_block_bytes bytes at block_ids[cb] * shard_block_bytes of members[r][m] live in the blob at
region_bases[m] + cb * shard_block_bytes * n_ranks + r * shard_block_bytes.
"""

from __future__ import annotations

import ctypes as C
from typing import Any, Sequence

from . import _native
from ._native import check, load


def _torch():
    import torch

    return torch


def _nbytes(t: Any) -> int:
    return t.numel() * t.element_size()


def _enable_peers(master: int, devices: set[int]) -> None:
    torch = _torch()
    lib = load()  # noqa: F841 - the library must be loaded before any op
    for d in devices:
        if d != master and not torch.cuda.can_device_access_peer(master, d):
            raise RuntimeError(f"device {master} cannot access peer device {d}")


def _member_arrays(members: Sequence[Sequence[Any]], shard_block_bytes: int):
    n_ranks, n_members = len(members), len(members[0])
    if any(len(r) != n_members for r in members):
        raise RuntimeError("every rank must provide the same members")
    flat = [members[r][m] for r in range(n_ranks) for m in range(n_members)]
    for i, t in enumerate(flat):
        if t.device.type != "cuda":
            raise RuntimeError("kvcache gather: tensor must be on device")
        if not t.is_contiguous():
            raise RuntimeError("kvcache gather: tensor must be contiguous")
    ptrs = (C.c_uint64 * len(flat))(*[t.data_ptr() for t in flat])
    sbb = (C.c_uint64 * n_members)(*([shard_block_bytes] * n_members))
    extent = (C.c_uint64 * n_members)(*[min(_nbytes(members[r][m]) for r in range(n_ranks)) for m in range(n_members)])
    return n_ranks, n_members, ptrs, sbb, extent, {t.device.index for t in flat}


def gather_tp_shards_to_chip(members: Sequence[Sequence[Any]], dst: Any, block_ids: Sequence[int],
                             shard_block_bytes: int, region_bases: Sequence[int],
                             header_words: Sequence[int] = (), blocking: bool = True) -> None:
    """Gather one chunk of a TP-sharded paged cache into `dst` on its GPU (see module doc)."""
    torch = _torch()
    n_ranks, n_members, ptrs, sbb, extent, devs = _member_arrays(members, shard_block_bytes)
    if len(region_bases) != n_members:
        raise RuntimeError(f"kvcache gather: {n_members} members but {len(region_bases)} region bases")
    master = dst.device.index
    _enable_peers(master, devs)
    ids = (C.c_uint32 * len(block_ids))(*block_ids)
    rb = (C.c_uint64 * n_members)(*region_bases)
    hw = (C.c_uint32 * max(1, len(header_words)))(*[int(w) & 0xFFFFFFFF for w in header_words])
    with torch.cuda.device(master):
        stream = torch.cuda.current_stream(master)
        check(load().kvs_gather_chunk(ptrs, n_ranks, n_members, sbb, extent, ids, len(block_ids), rb, hw,
                                      len(header_words), C.c_void_p(dst.data_ptr()), _nbytes(dst),
                                      C.c_void_p(stream.cuda_stream)))
        if blocking:
            stream.synchronize()


def scatter_chunk_from_chip(src: Any, members: Sequence[Sequence[Any]], block_ids: Sequence[int],
                            shard_block_bytes: int, region_bases: Sequence[int], blocking: bool = True) -> None:
    """Inverse of gather_tp_shards_to_chip: write each rank's slice of `src` into its blocks."""
    torch = _torch()
    n_ranks, n_members, ptrs, sbb, extent, devs = _member_arrays(members, shard_block_bytes)
    if len(region_bases) != n_members:
        raise RuntimeError(f"kvcache scatter: {n_members} members but {len(region_bases)} region bases")
    master = src.device.index
    _enable_peers(master, devs)
    ids = (C.c_uint32 * len(block_ids))(*block_ids)
    rb = (C.c_uint64 * n_members)(*region_bases)
    with torch.cuda.device(master):
        stream = torch.cuda.current_stream(master)
        check(load().kvs_scatter_chunk(C.c_void_p(src.data_ptr()), _nbytes(src), ptrs, n_ranks, n_members, sbb,
                                       extent, ids, len(block_ids), rb, C.c_void_p(stream.cuda_stream)))
        if blocking:
            stream.synchronize()


def pack_local_shards(members: Sequence[Any], dst: Any, block_ids: Sequence[int], shard_block_bytes: int,
                      region_bases: Sequence[int], header_words: Sequence[int] = (), blocking: bool = True) -> None:
    """Per-GPU pack: this GPU's own shard of every member into `dst` (one rank, no peers)."""
    gather_tp_shards_to_chip([list(members)], dst, block_ids, shard_block_bytes, region_bases, header_words, blocking)


def unpack_local_shards(src: Any, members: Sequence[Any], block_ids: Sequence[int], shard_block_bytes: int,
                        region_bases: Sequence[int], blocking: bool = True) -> None:
    scatter_chunk_from_chip(src, [list(members)], block_ids, shard_block_bytes, region_bases, blocking)


__all__ = ["gather_tp_shards_to_chip", "scatter_chunk_from_chip", "pack_local_shards", "unpack_local_shards",
           "paged_fill_cache_varlen", "paged_fill_cache_varlen_layers", "qk_norm_rope_fill",
           "paged_decode_attention", "evict_paged_kv"]
_ = _native


def paged_fill_cache_varlen(k_fill_value: Any, v_fill_value: Any, cu_seqlens: Any, page_table: Any,
                            start_positions: Any, cache_k: Any, cache_v: Any, out_of_range: Any = None):
    """Fill packed K/V of several requests into a paged KV cache, one token at a time.

    The B200 counterpart of ttnn.experimental.moreh_paged_fill_cache_varlen (patch 0002: kernels at
    lines 106-421, validation at 441-545), with its argument order and checks:
    k_fill_value / v_fill_value [1, num_kv_heads, total_tokens, head_dim]; cache_k / cache_v
    [max_num_blocks, num_kv_heads, block_size, head_dim] of the same dtype; cu_seqlens int32
    [batch_size + 1] (-1 after the valid offsets); page_table int32 [batch_size,
    max_num_blocks_per_seq]; start_positions int32 [batch_size]; every tensor a contiguous CUDA
    tensor on one device. Page-table entries <= 0 skip a token (vLLM's null block 0, -1 for unused
    slots). out_of_range: optional int32 CUDA tensor of one element, incremented for tokens skipped
    because their position or block is out of range. Asynchronous on the current stream; returns
    (cache_k, cache_v) as the reference's device operation does."""
    _check_fill(k_fill_value, v_fill_value, cu_seqlens, page_table, start_positions, cache_k, cache_v, out_of_range)
    torch = _torch()
    dev = k_fill_value.device
    heads, total, dim = k_fill_value.shape[1], k_fill_value.shape[2], k_fill_value.shape[3]
    P = C.c_void_p
    check(load().kvs_paged_fill_varlen(
        P(k_fill_value.data_ptr()), P(v_fill_value.data_ptr()), heads, total, dim * k_fill_value.element_size(),
        P(cu_seqlens.data_ptr()), page_table.shape[0], P(page_table.data_ptr()), page_table.shape[1],
        P(start_positions.data_ptr()), P(cache_k.data_ptr()), P(cache_v.data_ptr()), cache_k.shape[0],
        cache_k.shape[2], P(out_of_range.data_ptr() if out_of_range is not None else None),
        P(torch.cuda.current_stream(dev).cuda_stream)))
    return cache_k, cache_v


def _check_fill(k_fill_value, v_fill_value, cu_seqlens, page_table, start_positions, cache_k, cache_v,
                out_of_range) -> None:
    """The reference's validation of one fill (patch 0002 lines 441-545)."""
    torch = _torch()
    ts = {"k_fill_value": k_fill_value, "v_fill_value": v_fill_value, "cu_seqlens": cu_seqlens,
          "page_table": page_table, "start_positions": start_positions, "cache_k": cache_k, "cache_v": cache_v}
    for name, t in ts.items():
        if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
            raise RuntimeError(f"{name} must be on device!")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    dev = k_fill_value.device
    if any(t.device != dev for t in ts.values()):
        raise RuntimeError("All tensors must be on the same device!")
    if k_fill_value.dtype != cache_k.dtype:
        raise RuntimeError(f"k_fill_value dtype ({k_fill_value.dtype}) must match cache_k dtype ({cache_k.dtype})")
    if v_fill_value.dtype != cache_v.dtype:
        raise RuntimeError(f"v_fill_value dtype ({v_fill_value.dtype}) must match cache_v dtype ({cache_v.dtype})")
    if k_fill_value.dim() != 4 or cache_k.dim() != 4:
        raise RuntimeError("k_fill_value and cache_k must be 4-D")
    if k_fill_value.shape[0] != 1:
        raise RuntimeError(f"k_fill_value first dim must be 1, got {k_fill_value.shape[0]}")
    if v_fill_value.shape[0] != 1:
        raise RuntimeError(f"v_fill_value first dim must be 1, got {v_fill_value.shape[0]}")
    if k_fill_value.shape[-1] != cache_k.shape[-1]:
        raise RuntimeError("head_dim of k_fill_value must match cache_k")
    if v_fill_value.shape[-1] != cache_v.shape[-1]:
        raise RuntimeError("head_dim of v_fill_value must match cache_v")
    if k_fill_value.shape != v_fill_value.shape:
        raise RuntimeError("k_fill_value and v_fill_value must have the same shape")
    if cache_k.shape != cache_v.shape:
        raise RuntimeError("cache_k and cache_v must have the same shape")
    if k_fill_value.shape[1] != cache_k.shape[1]:
        raise RuntimeError("num_kv_heads of k_fill_value must match cache_k")
    for name in ("cu_seqlens", "page_table", "start_positions"):
        if ts[name].dtype != torch.int32:
            raise RuntimeError(f"{name} must be INT32")
    if page_table.dim() != 2:
        raise RuntimeError("page_table must be [batch_size, max_num_blocks_per_seq]")
    if page_table.shape[1] > cache_k.shape[0]:
        raise RuntimeError(f"max_num_blocks_per_seq ({page_table.shape[1]}) must be <= max_num_blocks ({cache_k.shape[0]})")
    if start_positions.shape[0] != page_table.shape[0]:
        raise RuntimeError(f"start_positions size ({start_positions.shape[0]}) must match batch_size ({page_table.shape[0]})")
    if cu_seqlens.numel() != page_table.shape[0] + 1:
        raise RuntimeError(f"cu_seqlens must hold batch_size + 1 = {page_table.shape[0] + 1} entries")
    if out_of_range is not None and (out_of_range.dtype != torch.int32 or out_of_range.device != dev):
        raise RuntimeError("out_of_range must be an int32 tensor on the fill's device")


def paged_fill_cache_varlen_layers(k_fill_values: Sequence[Any], v_fill_values: Sequence[Any], cu_seqlens: Any,
                                   page_table: Any, start_positions: Any, cache_ks: Sequence[Any],
                                   cache_vs: Sequence[Any], out_of_range: Any = None):
    """paged_fill_cache_varlen for several layers that share the requests and page tables, in one
    launch per 64 layers (no counterpart in the reference, which fills one layer per call). Layer
    l fills cache_ks[l] / cache_vs[l] from k_fill_values[l] / v_fill_values[l], every layer
    validated as the single-layer op validates it and of the first layer's shapes. Each layer's
    result equals the single-layer fill; out_of_range counts each skipped token once."""
    torch = _torch()
    n = len(k_fill_values)
    if not (len(v_fill_values) == len(cache_ks) == len(cache_vs) == n):
        raise RuntimeError("k_fill_values, v_fill_values, cache_ks and cache_vs must name the same layers")
    if n == 0:
        return cache_ks, cache_vs
    k0, c0 = k_fill_values[0], cache_ks[0]
    for l in range(n):
        _check_fill(k_fill_values[l], v_fill_values[l], cu_seqlens, page_table, start_positions, cache_ks[l],
                    cache_vs[l], out_of_range)
        if k_fill_values[l].shape != k0.shape or cache_ks[l].shape != c0.shape or cache_ks[l].dtype != c0.dtype:
            raise RuntimeError(f"layer {l}: every layer must have the first layer's shapes and dtype")
        if k_fill_values[l].device != k0.device:
            raise RuntimeError("All tensors must be on the same device!")
    heads, total, dim = k0.shape[1], k0.shape[2], k0.shape[3]
    P = C.c_void_p
    arr = lambda ts: (P * n)(*[t.data_ptr() for t in ts])
    check(load().kvs_paged_fill_varlen_layers(
        n, arr(k_fill_values), arr(v_fill_values), heads, total, dim * k0.element_size(),
        P(cu_seqlens.data_ptr()), page_table.shape[0], P(page_table.data_ptr()), page_table.shape[1],
        P(start_positions.data_ptr()), arr(cache_ks), arr(cache_vs), c0.shape[0], c0.shape[2],
        P(out_of_range.data_ptr() if out_of_range is not None else None),
        P(torch.cuda.current_stream(k0.device).cuda_stream)))
    return cache_ks, cache_vs


# ---------------------------------------------------------------- operators on a paged cache


def _dtype_code(dtype: Any) -> int:
    torch = _torch()
    return {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_FP16,
            torch.float8_e4m3fn: _native.DTYPE_E4M3}.get(dtype, -1)


def _on(device: Any, **tensors: Any) -> None:
    """Every tensor given (None: not given) is a CUDA tensor on `device` that needs no gradient and
    carries no tangent."""
    torch = _torch()
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
            raise RuntimeError(f"{name} must be on device!")
        if t.device != device:
            raise RuntimeError("All tensors must be on the same device!")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires grad, and the operators on a paged cache have no backward pass")
        if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} carries a tangent, and the operators on a paged cache have no derivatives")


def _int32(ndim: int, **tensors: Any) -> None:
    torch = _torch()
    for name, t in tensors.items():
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise RuntimeError(f"{name} must be INT32")
        if t.dim() != ndim or not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous, of {ndim} dimension(s)")


def _strides(t: Any, n: int, unit: int) -> list[int]:
    """Strides of the first n dimensions, `unit` bytes an element; a dimension of one element has none."""
    return [unit * s if size > 1 else 0 for size, s in zip(t.shape[:n], t.stride())]


def _rows(name: str, t: Any, ndim: int) -> None:
    if t.dim() != ndim:
        raise RuntimeError(f"{name} must be {ndim}-D")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise RuntimeError(f"{name} rows must be contiguous")


def _paged_cache(cache_k: Any, cache_v: Any, page_table: Any, k_scale: float, v_scale: float):
    """The C description of a layer's cache [num_blocks, num_kv_heads, block_size, head_dim], whose
    first three dimensions may have any strides (vLLM's [num_blocks, block_size, heads, head_dim] is
    passed as cache.transpose(1, 2))."""
    torch = _torch()
    if not isinstance(cache_k, torch.Tensor) or cache_k.device.type != "cuda":
        raise RuntimeError("cache_k must be on device!")
    _on(cache_k.device, cache_k=cache_k, cache_v=cache_v, page_table=page_table)
    _rows("cache_k", cache_k, 4)
    _rows("cache_v", cache_v, 4)
    if cache_k.shape != cache_v.shape or cache_k.dtype != cache_v.dtype:
        raise RuntimeError("cache_k and cache_v must have the same shape and dtype")
    _int32(2, page_table=page_table)
    code = _dtype_code(cache_k.dtype)
    if code < 0:
        raise RuntimeError(f"cache dtype ({cache_k.dtype}) must be bfloat16, float16 or float8_e4m3fn")
    blocks, heads, size, dim = cache_k.shape
    unit = cache_k.element_size()
    S3 = C.c_int64 * 3
    return _native.PagedCache(cache_k.data_ptr(), cache_v.data_ptr(), S3(*_strides(cache_k, 3, unit)),
                              S3(*_strides(cache_v, 3, unit)), page_table.data_ptr(), blocks, heads, size, dim,
                              page_table.shape[0], page_table.shape[1], code, k_scale, v_scale)


def _stream(device: Any):
    return C.c_void_p(_torch().cuda.current_stream(device).cuda_stream)


def _check_counter(t: Any) -> None:
    if t is not None and (t.dtype != _torch().int32 or t.numel() < 1):
        raise RuntimeError("out_of_range must be an int32 tensor of one element")


def _changed(*written: Any) -> None:
    """What a call has written counts as changed, so that autograd refuses a backward pass that saved
    it (tensors made in inference mode keep no count)."""
    for t in written:
        if t is not None and not t.is_inference():
            _torch().autograd.graph.increment_version(t)


def _ptr(t: Any):
    return None if t is None else t.data_ptr()


_S2 = C.c_int64 * 2


def _taken(done: Any) -> Any:
    """What the compiled entry returned; an error of a launch, which is not repeated, is its status."""
    if isinstance(done, int):
        check(done)
    return done


def qk_norm_rope_fill(q: Any, k: Any, v: Any, cos_sin: Any, cu_seqlens: Any, page_table: Any, start_positions: Any,
                      cache_k: Any, cache_v: Any, *, q_weight: Any = None, k_weight: Any = None, eps: float = 1e-6,
                      positions: Any = None, axes: Any = None, interleaved: bool = False, k_scale: float = 1.0,
                      v_scale: float = 1.0, q_out: Any = None, out_of_range: Any = None):
    """Per-head norms of queries and keys, rotation by the token's position and the fill of K and V
    into a paged cache, in one pass over q, k and v. Returns (q_out, cache_k, cache_v).

    q [tokens, q_heads, head_dim], k / v [tokens, num_kv_heads, head_dim]: bf16 or fp16, any strides
    with contiguous rows on 16-byte boundaries (slices of one projection's output, for example).
    cache_k / cache_v [num_blocks, num_kv_heads, block_size, head_dim] of the same dtype, or
    float8_e4m3fn holding value / k_scale and value / v_scale, any strides with contiguous rows.
    cu_seqlens, page_table and start_positions place the tokens as in paged_fill_cache_varlen.

    Per head x of q and k: x * weight / sqrt(mean(x^2) + eps) where q_weight / k_weight ([head_dim],
    the rows' dtype) is given, then the first cos_sin.shape[1] elements are rotated: pairs
    (i, i + rotary / 2), or (2i, 2i + 1) with interleaved. cos_sin: fp32 [positions, rotary], cosines of
    rotary / 2 frequencies, then their sines. A token's position is its position in the cache, or
    comes from positions: int32 [tokens], or [n_axes, tokens] (time, height and width of an image's
    tokens, say) with axes, int32 [rotary / 2], naming each frequency's axis. Computed in fp32 and
    rounded once.

    q_out may be q itself. A token whose slot is out of range stores no K and V; one whose position
    is outside cos_sin stores neither and gets a zero q_out row; out_of_range (int32, one element)
    counts both. Tokens behind the last sequence are left as they were in a given q_out and are zero
    in one allocated here. Two tokens must not share a slot. Asynchronous on the current stream."""
    fast = _native.opcall if _native.opcall is not None else _native.load_opcall()
    if fast:
        done = fast.fill(q, k, v, cos_sin, cu_seqlens, page_table, start_positions, cache_k, cache_v, q_weight, k_weight,
                         eps, positions, axes, interleaved, k_scale, v_scale, q_out, out_of_range)
        if done is not NotImplemented:
            return _taken(done), cache_k, cache_v
    torch = _torch()
    cache = _paged_cache(cache_k, cache_v, page_table, k_scale, v_scale)
    dev = cache_k.device
    _on(dev, q=q, k=k, v=v, cos_sin=cos_sin, cu_seqlens=cu_seqlens, start_positions=start_positions,
        q_weight=q_weight, k_weight=k_weight, positions=positions, axes=axes, q_out=q_out, out_of_range=out_of_range)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _rows(name, t, 3)
    tokens, q_heads, dim = q.shape
    if k.shape != v.shape or k.shape[0] != tokens or k.shape[1] != cache_k.shape[1]:
        raise RuntimeError("k and v must be [tokens, num_kv_heads, head_dim], with q's tokens and the cache's heads")
    if dim != cache_k.shape[3] or k.shape[2] != dim:
        raise RuntimeError("head_dim of q, k and v must match the cache")
    if not q.dtype == k.dtype == v.dtype:
        raise RuntimeError("q, k and v must have the same dtype")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and (t.shape != (dim,) or t.dtype != q.dtype or not t.is_contiguous()):
            raise RuntimeError(f"{name} must be a contiguous [head_dim] tensor of q's dtype")
    if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous():
        raise RuntimeError("cos_sin must be a contiguous float32 [positions, rotary] tensor")
    _int32(1, cu_seqlens=cu_seqlens, start_positions=start_positions, axes=axes)
    if start_positions.shape[0] != page_table.shape[0]:
        raise RuntimeError(f"start_positions size ({start_positions.shape[0]}) must match batch_size ({page_table.shape[0]})")
    if cu_seqlens.shape[0] != page_table.shape[0] + 1:
        raise RuntimeError(f"cu_seqlens must hold batch_size + 1 = {page_table.shape[0] + 1} entries")
    n_axes = 0
    if positions is not None:
        n_axes = positions.shape[0] if positions.dim() == 2 else 1
        _int32(positions.dim(), positions=positions)
        if positions.dim() not in (1, 2) or positions.shape[-1] != tokens or n_axes < 1:
            raise RuntimeError("positions must be [tokens] or [n_axes, tokens]")
    if axes is not None and axes.shape[0] * 2 != cos_sin.shape[1]:
        raise RuntimeError("axes must hold rotary / 2 entries")
    if axes is None and n_axes > 1:
        raise RuntimeError("positions of several axes need axes")
    _check_counter(out_of_range)
    zero_rest = q_out is None
    if q_out is None:
        q_out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=dev)
    else:
        _rows("q_out", q_out, 3)
        if q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise RuntimeError("q_out must have q's shape and dtype")
    rows = _native.QkvRows(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), _S2(*_strides(q, 2, 2)), _S2(*_strides(k, 2, 2)),
        _S2(*_strides(v, 2, 2)), _S2(*_strides(q_out, 2, 2)), cos_sin.data_ptr(), cu_seqlens.data_ptr(),
        start_positions.data_ptr(), _ptr(positions), _ptr(axes), _ptr(q_weight), _ptr(k_weight), _ptr(out_of_range),
        tokens, q_heads, cos_sin.shape[1], cos_sin.shape[0], n_axes, _dtype_code(q.dtype), eps, interleaved, zero_rest)
    check(load().kvs_qk_norm_rope_fill(C.byref(cache), C.byref(rows), _stream(dev)))
    _changed(cache_k, cache_v, None if zero_rest else q_out, out_of_range)
    return q_out, cache_k, cache_v


def _weight_sums(name: str, t: Any, batch: int, heads: int, cover: int) -> None:
    """A running sum of softmax weights: fp32 [batch, num_kv_heads, at least `cover` tokens]."""
    torch = _torch()
    if t.dtype != torch.float32 or t.dim() != 3 or t.stride(2) != 1 or t.shape[:2] != (batch, heads):
        raise RuntimeError(f"{name} must be float32 [batch_size, num_kv_heads, tokens] with contiguous rows")
    if t.shape[2] < cover:
        raise RuntimeError(f"{name} must cover max_num_blocks_per_seq * block_size = {cover} tokens")


def paged_decode_attention(q: Any, cache_k: Any, cache_v: Any, page_table: Any, seq_lens: Any, *,
                           scale: float | None = None, window: int | None = None, k_scale: float = 1.0,
                           v_scale: float = 1.0, out: Any = None, return_lse: bool = False, weights: Any = None,
                           weights_out: Any = None):
    """Attention of one new token per request over its paged K / V cache.

    q [batch, q_heads, head_dim] (bf16 or fp16, any strides with contiguous rows on 16-byte boundaries);
    query head g reads KV head g // (q_heads // num_kv_heads). cache_k / cache_v / k_scale / v_scale as
    in qk_norm_rope_fill; page_table int32 [batch, max_num_blocks_per_seq]; seq_lens int32 [batch], the
    new token included (its K and V are in the cache). Request b attends to the tokens below seq_lens[b]
    that have a page (entry > 0), the last `window` of them where given, with scale (head_dim ** -0.5 if
    None) on the scores. A request without tokens gets zeros and a log-sum-exp of -inf. Returns out
    [batch, q_heads, head_dim], or (out, lse) with lse fp32 [batch, q_heads].

    weights (fp32 [batch, num_kv_heads, tokens], covering the page table's tokens) accumulates what
    evict_paged_kv chooses by: weights_out (default: weights itself) becomes weights plus each token's
    softmax weight summed over the KV head's query heads, for the tokens below seq_lens. Such a call
    allocates 4 bytes for each query head and token of the page table (64 requests, 64 query heads and rows
    of 131072 tokens: 2 GiB), whatever the lengths are: cut page_table and weights to the longest context.
    Equal calls give equal bits. Asynchronous on the current stream; no backward pass."""
    fast = _native.opcall if _native.opcall is not None else _native.load_opcall()
    if fast:
        done = fast.attend(q, cache_k, cache_v, page_table, seq_lens, scale, window, k_scale, v_scale, out, return_lse,
                           weights, weights_out)
        if done is not NotImplemented:
            return _taken(done)
    torch = _torch()
    cache = _paged_cache(cache_k, cache_v, page_table, k_scale, v_scale)
    dev = cache_k.device
    _on(dev, q=q, seq_lens=seq_lens, out=out, weights=weights, weights_out=weights_out)
    _rows("q", q, 3)
    batch, q_heads, dim = q.shape
    if batch != page_table.shape[0] or dim != cache_k.shape[3]:
        raise RuntimeError("q must be [batch_size, q_heads, head_dim] of the page table's requests and the cache's head_dim")
    _int32(1, seq_lens=seq_lens)
    if seq_lens.shape[0] != batch:
        raise RuntimeError(f"seq_lens size ({seq_lens.shape[0]}) must match batch_size ({batch})")
    if window is not None and not 0 < window < 1 << 31:
        raise RuntimeError("window must be 1 to 2^31 - 1 tokens")
    given = out
    if out is None:
        out = torch.empty((batch, q_heads, dim), dtype=q.dtype, device=dev)
    else:
        _rows("out", out, 3)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise RuntimeError("out must have q's shape and dtype")
    rows = _native.DecodeRows(q.data_ptr(), out.data_ptr(), _S2(*_strides(q, 2, 2)), _S2(*_strides(out, 2, 2)),
                              seq_lens.data_ptr())
    rows.q_heads, rows.dtype = q_heads, _dtype_code(q.dtype)
    rows.window = window or 0
    rows.scale = dim ** -0.5 if scale is None else scale
    lse = None
    if return_lse:
        lse = torch.empty((batch, q_heads), dtype=torch.float32, device=dev)
        rows.lse = lse.data_ptr()
    if weights is not None:
        weights_out = weights if weights_out is None else weights_out
        cover = page_table.shape[1] * cache_k.shape[2]
        _weight_sums("weights", weights, batch, cache_k.shape[1], cover)
        _weight_sums("weights_out", weights_out, batch, cache_k.shape[1], cover)
        rows.weights, rows.weights_out = weights.data_ptr(), weights_out.data_ptr()
        rows.weights_strides = _S2(*_strides(weights, 2, 1))
        rows.weights_out_strides = _S2(*_strides(weights_out, 2, 1))
        rows.w_len = min(weights.shape[2], weights_out.shape[2])
    elif weights_out is not None:
        raise RuntimeError("weights_out needs weights")
    lib = load()
    need = C.c_uint64()
    check(lib.kvs_decode_attention_workspace(C.byref(cache), C.byref(rows), dev.index, C.byref(need)))
    workspace = torch.empty(need.value, dtype=torch.uint8, device=dev)
    rows.workspace, rows.workspace_bytes = workspace.data_ptr(), need.value
    check(lib.kvs_paged_decode_attention(C.byref(cache), C.byref(rows), _stream(dev)))
    _changed(given, weights_out)
    return (out, lse) if return_lse else out


def evict_paged_kv(cache_k: Any, cache_v: Any, page_table: Any, seq_lens: Any, weights: Any, keep: int, *,
                   first: int = 0, recent: int = 0, dst_page_table: Any = None, weights_out: Any = None,
                   out_of_range: Any = None):
    """Trim paged caches to the tokens that attention reads most. Returns (kept, new_lens).

    Per request and KV head, of the tokens below seq_lens that have a page: the first `first` and the
    last `recent` positions stay, and of the others those of the largest weight (equal weights: the
    lowest position; NaN counts as the largest), `keep` in all. kept: int32 [batch, num_kv_heads, keep],
    the kept positions in order, then -1; new_lens: int32 [batch], min(keep, tokens).

    The kept rows move in order to slots 0, 1, ... of dst_page_table (int32 [batch, blocks], covering
    keep slots), fresh pages that no table of the call reads, so pages shared between requests or held
    by a store stay as they are. Without dst_page_table (or with page_table itself) they move within the
    request's own pages, which then no other request may share, nor name one page twice. A slot without a valid page stores
    nothing and is counted in out_of_range (int32, one element). weights: fp32 [batch, num_kv_heads,
    tokens] as paged_decode_attention accumulates them, covering the page table's tokens; weights_out
    (default: weights itself) receives the kept tokens' weights, then zeros up to seq_lens. Keys keep the
    rotation of their old positions: rotate new tokens by the `positions` of qk_norm_rope_fill.
    Asynchronous on the current stream."""
    fast = _native.opcall if _native.opcall is not None else _native.load_opcall()
    if fast:
        done = fast.evict(cache_k, cache_v, page_table, seq_lens, weights, keep, first, recent, dst_page_table,
                          weights_out, out_of_range)
        if done is not NotImplemented:
            return _taken(done)
    torch = _torch()
    cache = _paged_cache(cache_k, cache_v, page_table, 1.0, 1.0)
    dev = cache_k.device
    weights_out = weights if weights_out is None else weights_out
    _on(dev, seq_lens=seq_lens, weights=weights, dst_page_table=dst_page_table, weights_out=weights_out,
        out_of_range=out_of_range)
    _int32(1, seq_lens=seq_lens)
    _int32(2, dst_page_table=dst_page_table)
    batch, heads = page_table.shape[0], cache_k.shape[1]
    if seq_lens.shape[0] != batch:
        raise RuntimeError(f"seq_lens size ({seq_lens.shape[0]}) must match batch_size ({batch})")
    if dst_page_table is not None and dst_page_table.shape[0] != batch:
        raise RuntimeError(f"dst_page_table must have batch_size ({batch}) rows")
    if dst_page_table is not None and dst_page_table.shape[1] < 1:
        raise RuntimeError(f"dst_page_table must cover keep ({keep}) slots")
    if keep <= 0 or keep >= 1 << 31 or first < 0 or recent < 0 or first + recent > keep:
        raise RuntimeError(f"keep ({keep}) must be 1 to 2^31 - 1, first ({first}) and recent ({recent}) not negative and "
                           "first + recent <= keep")
    cover = page_table.shape[1] * cache_k.shape[2]
    _weight_sums("weights", weights, batch, heads, cover)
    _weight_sums("weights_out", weights_out, batch, heads, cover)
    _check_counter(out_of_range)
    kept = torch.empty((batch, heads, keep), dtype=torch.int32, device=dev)
    new_lens = torch.empty((batch,), dtype=torch.int32, device=dev)
    rows = _native.EvictRows(
        seq_lens.data_ptr(), _ptr(dst_page_table), weights.data_ptr(),
        weights_out.data_ptr(), _S2(*_strides(weights, 2, 1)), _S2(*_strides(weights_out, 2, 1)), kept.data_ptr(),
        new_lens.data_ptr(), _ptr(out_of_range), 0 if dst_page_table is None else dst_page_table.shape[1], weights.shape[2],
        weights_out.shape[2], keep, first, recent)
    check(load().kvs_evict_paged(C.byref(cache), C.byref(rows), _stream(dev)))
    _changed(cache_k, cache_v, weights_out, out_of_range)
    return kept, new_lens
