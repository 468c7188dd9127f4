"""The operators around the paged KV cache, as they are measured: their cases, inputs and plain forms.

Three operators work on one set of pages, as a decode step uses them:

* fill   -- norms of queries and keys per head, rotation by the token's position (one or several
            axes), and the write of K and V into the paged cache (`ops.qk_norm_rope_fill`);
* attend -- attention of one new token per request over the paged cache, optionally adding each
            token's softmax weight to a running sum (`ops.paged_decode_attention`);
* evict  -- keeping, per request and KV head, the tokens of the largest accumulated weight and
            moving their rows to fresh pages (`ops.evict_paged_kv`).

`run` computes them in elementary torch operations in 32 bits, or, where `own` is set, by the
package's kernels on the same state. `exact` computes the definitions in 64 bits.
"""

import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0


def listed():
    fill = dict(op="fill", kv_heads=8, q_heads=64, head_dim=128, rotary=128, page=64, dtype="bf16", cache="same",
                layout="hnd", norm=True, axes=1, interleaved=False, pad=0)
    attend = dict(op="attend", kv_heads=8, group=8, head_dim=128, page=64, dtype="bf16", cache="same", layout="hnd",
                  window=0, weights=False)
    evict = dict(op="evict", kv_heads=8, head_dim=128, page=64, dtype="bf16", layout="hnd", first=4, recent=64)
    return [
        # the token step of one request: latency only
        dict(fill, name="fill_token", requests=1, tokens=1, mix=1),
        # the token step of a full decode batch, its last rows padding of a captured graph
        dict(fill, name="fill_batch_tokens", requests=120, tokens=120, pad=8, mix=2),
        # chunked prefill of four requests, 8192 tokens, one Qwen3-32B layer
        dict(fill, name="fill_prefill", requests=4, tokens=8192, mix=3),
        # image and text tokens with time / height / width positions into an fp8 cache, token-major pages
        dict(fill, name="fill_axes_fp8", requests=7, tokens=5001, q_heads=32, kv_heads=4, axes=3, cache="fp8",
             layout="nhd", page=16, pad=23, mix=4),
        # the first steps of a chat: short contexts, latency only
        dict(attend, name="attend_short", batch=2, max_len=193, mix=5),
        # one request with a long document
        dict(attend, name="attend_long", batch=1, max_len=131071, mix=6),
        # a serving batch of mixed lengths
        dict(attend, name="attend_batch", batch=48, max_len=16384, mix=7),
        # the same from an fp8 cache in token-major pages of 16
        dict(attend, name="attend_fp8", batch=64, max_len=12001, cache="fp8", layout="nhd", page=16, mix=8),
        # fp16, smaller heads and group, a sliding window
        dict(attend, name="attend_window", batch=33, max_len=9001, dtype="fp16", head_dim=64, group=5, window=4096,
             page=32, mix=9),
        # decode that also sums each token's weight, for the eviction below
        dict(attend, name="attend_weights", batch=16, max_len=8192, weights=True, mix=10),
        # one request trimmed back to its budget
        dict(evict, name="evict_one", batch=1, max_len=4200, keep=2048, mix=11),
        # long prompts compressed after prefill
        dict(evict, name="evict_batch", batch=12, max_len=32768, keep=4096, mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One case of the ranges that the listed ones stand for."""
    op = rng.choice(["fill", "attend", "evict"])
    common = dict(op=op, kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 80, 96, 128, 128, 256]),
                  page=rng.choice([16, 32, 48, 64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                  layout=rng.choice(["hnd", "nhd"]), mix=rng.randrange(1 << 30))
    row = common["kv_heads"] * common["head_dim"]
    if op == "fill":
        tokens = _log(rng, 1, 8192)
        group = rng.choice([1, 4, 7, 8])
        while row * (group + 2) * tokens > 80 * 128 * 8192:
            tokens //= 2
        tokens = max(1, tokens)
        requests = tokens if rng.random() < 0.3 and tokens <= 256 else max(1, min(tokens, rng.randint(1, 40)))
        rotary = rng.choice([common["head_dim"], common["head_dim"] // 16 * 8])
        return dict(common, requests=requests, tokens=tokens, q_heads=common["kv_heads"] * group, rotary=rotary,
                    cache=rng.choice(["same", "same", "fp8"]), norm=rng.random() < 0.7, axes=rng.choice([1, 1, 3]),
                    interleaved=rng.random() < 0.3, pad=rng.choice([0, 0, rng.randint(1, 40)]))
    most = 8 * 128 * 16384 * 48
    if op == "attend":
        batch, max_len = _log(rng, 1, 160), _log(rng, 1, 131072)
        while batch * max_len * row > most:
            batch, max_len = max(1, batch // 2), max(1, max_len * 3 // 4)
        return dict(common, batch=batch, max_len=max_len, group=rng.choice([1, 4, 5, 8, 8, 16]),
                    cache=rng.choice(["same", "same", "fp8"]),
                    window=rng.choice([0, 0, rng.randint(1, max(1, max_len))]), weights=rng.random() < 0.3)
    batch, max_len = _log(rng, 1, 48), _log(rng, 2, 65536)
    while batch * max_len * row > most // 4:
        batch, max_len = max(1, batch // 2), max(2, max_len * 3 // 4)
    keep = rng.randint(1, max_len)
    first = min(4, keep // 4)
    return dict(common, batch=batch, max_len=max_len, keep=keep, first=first, recent=rng.randint(0, (keep - first) // 2))


# ------------------------------------------------------------------ what a case fixes (not the seed)


def _lengths(case):
    """Context lengths of an attend or evict case: the longest one, then a spread of shorter ones;
    larger batches end with an empty row, the padding of a captured decode graph."""
    r = random.Random(case["mix"])
    n, top = case["batch"], case["max_len"]
    lens = [top] + [r.randint(max(1, top // 8), top) for _ in range(n - 1)]
    if n >= 8:
        lens[-1] = 0
    return lens


def _pieces(case):
    """(tokens, start position) of every request of a fill case."""
    r = random.Random(case["mix"])
    n, total = case["requests"], case["tokens"]
    cuts = sorted(r.sample(range(1, total), n - 1)) if n > 1 else []
    lens = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return [(c, r.choice([0, r.randint(0, 700)])) for c in lens]


def _element(case):
    return 1 if case.get("cache") == "fp8" else 2


def work(case):
    d, kv, el = case["head_dim"], case["kv_heads"], _element(case)
    if case["op"] == "fill":
        t = case["tokens"]
        rows = case["q_heads"] + 2 * kv
        read = 2 * t * rows * d + 4 * t * case["rotary"]
        wrote = 2 * t * case["q_heads"] * d + el * t * 2 * kv * d
        return {"bytes": read + wrote, "flops": t * (case["q_heads"] + kv) * d * 8}
    lens = _lengths(case)
    if case["op"] == "attend":
        seen = [min(x, case["window"]) if case["window"] else x for x in lens]
        heads = kv * case["group"]
        pages = sum(-(-x // case["page"]) for x in seen)
        nbytes = el * 2 * kv * d * sum(seen) + 4 * len(lens) * heads * d + 4 * len(lens) * heads + 4 * pages
        if case["weights"]:
            nbytes += 8 * kv * sum(lens)
        return {"bytes": nbytes, "flops": 4 * heads * d * sum(seen)}
    kept = sum(min(x, case["keep"]) for x in lens)
    return {"bytes": kv * (4 * sum(lens) + kept * (2 * 2 * 2 * d + 4 + 4)), "flops": kv * sum(lens)}


# ------------------------------------------------------------------ inputs


def _tables(g, pages_of, width, extra):
    """Page tables of requests with the given page counts over a pool of shuffled pages; page 0 is
    the null page, unused entries are -1. Returns (table on the GPU, pages in the pool)."""
    total = sum(pages_of)
    ids = torch.randperm(total + extra, generator=g, device="cuda")[:total] + 1
    table = torch.full((len(pages_of), max(1, width)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = ids[at:at + n].to(torch.int32)
        at += n
    return table, total + extra + 1


def _cache(g, case, pages):
    """A cache [pages, kv_heads, page, head_dim]; `nhd` pages are token-major in memory."""
    h, n, d = case["kv_heads"], case["page"], case["head_dim"]
    shape = (pages, h, n, d) if case["layout"] == "hnd" else (pages, n, h, d)
    t = torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=g)
    if case.get("cache") == "fp8":
        t = (t / 0.05).clamp(-FP8_MAX, FP8_MAX).to(FP8)
    return t if case["layout"] == "hnd" else t.transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    kv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    s = {"op": case["op"], "case": case}
    # fp8 caches hold value / scale
    s["k_scale"], s["v_scale"] = (0.05, 0.05) if case.get("cache") == "fp8" else (1.0, 1.0)
    if case["op"] == "fill":
        pieces = _pieces(case)
        t, hq = case["tokens"] + case["pad"], case["q_heads"]
        # q, k, v are slices of one projection's output
        qkv = torch.empty((t, (hq + 2 * kv) * d), dtype=dt, device="cuda").normal_(generator=g)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, kv * d, kv * d], dim=1))
        last = max(c + p for c, p in pieces)
        pages_of = [-(-(c + p) // page) for c, p in pieces]
        s["page_table"], pages = _tables(g, pages_of, max(pages_of), 3)
        s["cache_k"], s["cache_v"] = _cache(g, case, pages), _cache(g, case, pages)
        s["cu_seqlens"] = torch.tensor([0] + [c for c, _ in pieces], device="cuda").cumsum(0).to(torch.int32)
        s["start_positions"] = torch.tensor([p for _, p in pieces], dtype=torch.int32, device="cuda")
        half = case["rotary"] // 2
        freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = torch.arange(last + 64, dtype=torch.float64, device="cuda")[:, None] * freq
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        s["q_weight"] = s["k_weight"] = s["positions"] = s["axes"] = None
        if case["norm"]:
            s["q_weight"], s["k_weight"] = ((1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in "qk")
        if case["axes"] > 1:  # an image's tokens share a time step and differ in row and column
            s["positions"] = torch.randint(0, last + 64, (case["axes"], t), generator=g, device="cuda").to(torch.int32)
            s["axes"] = (torch.arange(half, device="cuda") * case["axes"] // half).to(torch.int32)
        return s
    lens = _lengths(case)
    pages_of = [-(-x // page) for x in lens]
    new = [-(-min(x, case["keep"]) // page) for x in lens] if case["op"] == "evict" else []
    table, pages = _tables(g, pages_of + new, max(pages_of + [1]), 2)
    s["page_table"] = table[:len(lens)].contiguous()
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["cache_k"], s["cache_v"] = _cache(g, case, pages), _cache(g, case, pages)
    width = s["page_table"].shape[1] * page
    weights = None
    if case["op"] == "evict" or case["weights"]:
        # sums of softmax weights: a few large, many small, some never attended (equal, zero)
        weights = (torch.empty((len(lens), kv, width), device="cuda").normal_(generator=g) * 2).exp()
        weights *= torch.rand(weights.shape, generator=g, device="cuda") > 0.1
        weights *= torch.arange(width, device="cuda") < s["seq_lens"][:, None, None]
    s["weights"] = weights
    if case["op"] == "attend":
        s["q"] = torch.empty((len(lens), kv * case["group"], d), dtype=dt, device="cuda").normal_(generator=g) * 2
        s["weights_out"] = torch.zeros_like(weights) if weights is not None else None
        s["scale"] = d ** -0.5
    else:
        s["dst_page_table"] = table[len(lens):, :max(1, -(-case["keep"] // page))].contiguous()
        s["weights_out"] = torch.zeros_like(weights)
    return s


# ------------------------------------------------------------------ one pass


def _ops():
    if "tt-infinity_b200" not in sys.path:
        sys.path.insert(1, "tt-infinity_b200")
    from kvcache_manager import ops

    return ops


def run(s):
    if own:
        return _own(s)
    return {"fill": _plain_fill, "attend": _plain_attend, "evict": _plain_evict}[s["op"]](s)


def _own(s):
    ops, c = _ops(), s["case"]
    if s["op"] == "fill":
        q, ck, cv = ops.qk_norm_rope_fill(
            s["q"], s["k"], s["v"], s["cos_sin"], s["cu_seqlens"], s["page_table"], s["start_positions"], s["cache_k"],
            s["cache_v"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6, positions=s["positions"],
            axes=s["axes"], interleaved=c["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"q": q, "cache_k": ck, "cache_v": cv}
    if s["op"] == "attend":
        out, lse = ops.paged_decode_attention(
            s["q"], s["cache_k"], s["cache_v"], s["page_table"], s["seq_lens"], scale=s["scale"],
            window=c["window"] or None, k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True,
            weights=s["weights"], weights_out=s["weights_out"])
        return {"out": out, "lse": lse, "weights": s["weights_out"]}
    kept, lens = ops.evict_paged_kv(
        s["cache_k"], s["cache_v"], s["page_table"], s["seq_lens"], s["weights"], c["keep"], first=c["first"],
        recent=c["recent"], dst_page_table=s["dst_page_table"], weights_out=s["weights_out"])
    return {"kept": kept, "lens": lens, "cache_k": s["cache_k"], "cache_v": s["cache_v"], "weights": s["weights_out"]}


def _rotate(x, cos, sin, interleaved):
    """x [tokens, heads, rotary] rotated by the tokens' cos and sin [tokens, 1, rotary / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _store(cache, pages, rows, write, values):
    """cache[pages[t], :, rows[t]] = values[t] where write[t]; other tokens leave the cache as it was."""
    raw = cache.view(torch.uint8) if cache.dtype == FP8 else cache
    if cache.dtype == FP8:
        values = values.clamp(-FP8_MAX, FP8_MAX).to(FP8).view(torch.uint8)
    old = raw[pages, :, rows]
    raw[pages, :, rows] = torch.where(write[:, None, None], values.to(raw.dtype), old)


def _plain_fill(s):
    c = s["case"]
    t = torch.arange(s["q"].shape[0], device="cuda")
    ends = s["cu_seqlens"][1:].long()
    live = t < ends[-1]
    req = torch.searchsorted(ends, t, right=True).clamp(max=ends.numel() - 1)
    slot = t - s["cu_seqlens"].long()[req] + s["start_positions"].long()[req]
    slot = torch.where(live, slot, 0)
    page = s["page_table"].long()[req, slot // c["page"]]
    write = live & (page > 0)
    half = c["rotary"] // 2
    if s["positions"] is None:
        angles = s["cos_sin"][slot]
        cos, sin = angles[:, None, :half], angles[:, None, half:]
    else:
        pos = s["positions"].long()[s["axes"].long()].T  # [tokens, half]
        i = torch.arange(half, device="cuda")
        cos, sin = s["cos_sin"][pos, i][:, None], s["cos_sin"][pos, i + half][:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        r = c["rotary"]
        return torch.cat([_rotate(x[..., :r], cos, sin, c["interleaved"]), x[..., r:]], dim=-1)

    q = torch.where(live[:, None, None], turned(s["q"], s["q_weight"]), 0).to(s["q"].dtype)
    page, row = torch.where(write, page, 0), slot % c["page"]
    _store(s["cache_k"], page, row, write, turned(s["k"], s["k_weight"]) / s["k_scale"])
    _store(s["cache_v"], page, row, write, s["v"].float() / s["v_scale"])
    return {"q": q, "cache_k": s["cache_k"], "cache_v": s["cache_v"]}


def _rows(cache, table):
    """The cache's rows in the order of the page table, in 32 bits: [batch, kv_heads, tokens, head_dim]."""
    raw = cache.view(torch.uint8) if cache.dtype == FP8 else cache
    x = raw[table.long().clamp(min=0)]
    return (x.view(FP8) if cache.dtype == FP8 else x).float().transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    c = s["case"]
    k = _rows(s["cache_k"], s["page_table"])
    b, kv, n, d = k.shape
    t = torch.arange(n, device="cuda")
    lens = s["seq_lens"][:, None]
    seen = (t < lens) & (s["page_table"] > 0).repeat_interleave(c["page"], dim=1)
    if c["window"]:
        seen = seen & (t >= lens - c["window"])
    seen = seen[:, None, None]
    q = s["q"].float().view(b, kv, c["group"], d)
    score = torch.matmul(q, k.transpose(2, 3)) * (s["scale"] * s["k_scale"])
    del k
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)
    v = _rows(s["cache_v"], s["page_table"])
    v = torch.where(seen[:, 0, 0, None, :, None], v, 0)
    out = torch.matmul(p, v) * s["v_scale"]
    lse = (top + total.log()).reshape(b, kv * c["group"])
    if s["weights"] is not None:
        s["weights_out"].copy_(torch.where((t < lens)[:, None], s["weights"] + p.sum(2), s["weights_out"]))
    return {"out": out.reshape(b, kv * c["group"], d).to(s["q"].dtype), "lse": lse, "weights": s["weights_out"]}


def _plain_evict(s):
    c = s["case"]
    w, lens, keep, page = s["weights"], s["seq_lens"].long()[:, None, None], c["keep"], c["page"]
    n = w.shape[2]
    t = torch.arange(n, device="cuda")
    there = (t < lens) & (s["page_table"] > 0).repeat_interleave(page, dim=1)[:, None]
    bound = there & ((t < c["first"]) | (t >= lens - c["recent"]))
    key = torch.where(bound, math.inf, torch.where(there, w, -math.inf))
    width = min(keep, n)
    order = torch.sort(key, dim=2, descending=True, stable=True).indices[..., :width]
    count = there.sum(-1, keepdim=True).clamp(max=keep)  # [batch, 1, 1]
    i = torch.arange(width, device="cuda")
    at = torch.where(i < count, order, n).sort(dim=2).values
    live = i < count
    kept = torch.full((*w.shape[:2], keep), -1, dtype=torch.int32, device="cuda")
    kept[..., :width] = torch.where(live, at, -1)
    at = torch.where(live, at, 0)
    b = torch.arange(w.shape[0], device="cuda")[:, None, None]
    h = torch.arange(w.shape[1], device="cuda")[:, None]
    src_page, src_row = s["page_table"].long()[b, at // page].clamp(min=0), at % page
    dst_page, dst_row = s["dst_page_table"].long()[:, i // page][:, None].clamp(min=0), i % page

    def move(cache):
        rows = torch.where(live[..., None], cache[src_page, h, src_row], cache[dst_page, h, dst_row])
        cache[dst_page, h, dst_row] = rows

    move(s["cache_k"])
    move(s["cache_v"])
    s["weights_out"].zero_()
    s["weights_out"][..., :width] = torch.where(live, w.gather(2, at), 0)
    return {"kept": kept, "lens": count[:, 0, 0].to(torch.int32), "cache_k": s["cache_k"], "cache_v": s["cache_v"],
            "weights": s["weights_out"]}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    """What `run` returns, from the definitions, one request at a time in 64 bits."""
    s = prepare(case, seed)
    return {"fill": _exact_fill, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](case, s)


def _slots(case, table, b, positions):
    """(page, row) of request b's positions."""
    return table[b, torch.div(positions, case["page"], rounding_mode="floor")].long(), positions % case["page"]


def _exact_fill(case, s):
    half, r = case["rotary"] // 2, case["rotary"]
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    ck, cv = s["cache_k"].double(), s["cache_v"].double()
    index = torch.arange(half, device="cuda")
    at = 0
    for b, (count, start) in enumerate(_pieces(case)):
        tok = slice(at, at + count)
        at += count
        position = start + torch.arange(count, device="cuda")
        page, row = _slots(case, s["page_table"], b, position)
        if case["axes"] > 1:
            by_frequency = torch.stack([s["positions"][int(a), tok].long() for a in s["axes"].tolist()], dim=1)
        else:
            by_frequency = position[:, None].expand(count, half)
        turn = torch.complex(s["cos_sin"].double()[by_frequency, index], s["cos_sin"].double()[by_frequency, index + half])

        def rows(x, weight):
            y = x[tok].double()
            if weight is not None:
                y = y / torch.sqrt(torch.linalg.vecdot(y, y)[..., None] / y.shape[-1] + 1e-6) * weight.double()
            z = y.clone()
            first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, half), slice(half, r))
            turned = torch.complex(y[..., first], y[..., second]) * turn[:, None]
            z[..., first], z[..., second] = turned.real, turned.imag
            return z

        q[tok] = rows(s["q"], s["q_weight"])
        ck[page, :, row] = rows(s["k"], s["k_weight"]) / s["k_scale"]
        cv[page, :, row] = s["v"][tok].double() / s["v_scale"]
    if case["cache"] == "fp8":  # an 8-bit cache holds nothing beyond its largest value
        ck.clamp_(-FP8_MAX, FP8_MAX)
        cv.clamp_(-FP8_MAX, FP8_MAX)
    return {"q": q, "cache_k": ck, "cache_v": cv}


def _exact_attend(case, s):
    kv, g, d = case["kv_heads"], case["group"], case["head_dim"]
    lens = _lengths(case)
    out = torch.zeros((len(lens), kv * g, d), dtype=torch.float64, device="cuda")
    lse = torch.full((len(lens), kv * g), -math.inf, dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights_out"].double()
    for b, n in enumerate(lens):
        if weights is not None:
            weights[b, :, :n] = s["weights"][b, :, :n].double()
        low = max(0, n - case["window"]) if case["window"] else 0
        if low >= n:
            continue
        page, row = _slots(case, s["page_table"], b, torch.arange(low, n, device="cuda"))
        for h in range(kv):
            k = s["cache_k"][:, h].view(torch.uint8 if s["cache_k"].dtype == FP8 else s["cache_k"].dtype)[page, row]
            v = s["cache_v"][:, h].view(torch.uint8 if s["cache_v"].dtype == FP8 else s["cache_v"].dtype)[page, row]
            k, v = (x.view(FP8).double() if s["cache_k"].dtype == FP8 else x.double() for x in (k, v))
            heads = slice(h * g, h * g + g)
            score = k @ s["q"][b, heads].double().T * (s["scale"] * s["k_scale"])
            lse[b, heads] = torch.logsumexp(score, 0)
            p = (score - lse[b, heads]).exp()
            out[b, heads] = p.T @ v * s["v_scale"]
            if weights is not None:
                weights[b, h, low:n] += p.sum(1)
    return {"out": out, "lse": lse, "weights": weights}


def _exact_evict(case, s):
    kv, keep = case["kv_heads"], case["keep"]
    lens = _lengths(case)
    ck, cv = s["cache_k"].clone(), s["cache_v"].clone()
    kept = torch.full((len(lens), kv, keep), -1, dtype=torch.int32, device="cuda")
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        m = min(n, keep)
        to_page, to_row = _slots(case, s["dst_page_table"], b, torch.arange(m, device="cuda"))
        for h in range(kv):
            w = s["weights"][b, h, :n].tolist()
            always = set(range(min(case["first"], n))) | set(range(max(0, n - case["recent"]), n))
            rest = sorted((i for i in range(n) if i not in always), key=lambda i: (-w[i], i))
            chosen = sorted(list(always) + rest[:max(0, m - len(always))]) if n > keep else list(range(n))
            at = torch.tensor(chosen, dtype=torch.long, device="cuda")
            kept[b, h, :m] = at.to(torch.int32)
            weights[b, h, :m] = s["weights"][b, h, at].double()
            page, row = _slots(case, s["page_table"], b, at)
            ck[to_page, h, to_row] = s["cache_k"][page, h, row]
            cv[to_page, h, to_row] = s["cache_v"][page, h, row]
    return {"kept": kept, "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32, device="cuda"),
            "cache_k": ck.double(), "cache_v": cv.double(), "weights": weights}
