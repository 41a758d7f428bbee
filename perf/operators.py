"""Cases of the 8-bit KV cache operators: rotary positions with several axes, the cache's write, read-back and eviction, and paged attention over it.

``own`` False computes each operator in plain torch (fp32, rounded once at the end), True calls the framework.
A cache is four tensors: codes ``k_cache`` / ``v_cache`` [num_blocks, kv_heads, block_size, head_dim] (int8 or float8_e4m3fn) and scales
``k_scale`` / ``v_scale`` [num_blocks, kv_heads, block_size / group] (float32); an element's value is code * scale.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = 2.0 ** -100  # a group whose largest magnitude is below this is held as zeros


# ----------------------------------------------------------------------------- cases
def _rotary(name, tokens, q_heads, kv_heads, head_dim, rot_dim, axes, interleaved, inverse, dtype):
    return dict(name=name, op="rotary", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rot_dim=rot_dim, axes=axes,
                interleaved=interleaved, inverse=inverse, dtype=dtype)


def _cache(name, op, seqs, context, kv_heads, head_dim, block_size, group, cache, dtype, **more):
    return dict(name=name, op=op, seqs=seqs, context=context, kv_heads=kv_heads, head_dim=head_dim, block_size=block_size, group=group,
                cache=cache, dtype=dtype, **more)


def listed():
    return [
        # one decode step of 64 requests: 32 / 8 heads of 128, three axes (time, height, width)
        _rotary("rotary_step", 64, 32, 8, 128, 128, 3, False, False, "bf16"),
        # the gradient form over a long prompt of images: two axes, part of each head rotated, an odd number of tokens
        _rotary("rotary_images_inverse", 16381, 32, 8, 128, 96, 2, True, True, "fp16"),
        # one decode step's append: 64 requests with contexts up to 8192, pages of 128
        _cache("write_step", "write", 64, 8191, 8, 128, 128, 16, "e4m3", "bf16", tokens=1),
        # prompts of ragged length, most of them new, some that continue a cached prefix; read back whole as 16-bit rows
        _cache("write_prompts", "write", 16, 500, 8, 128, 128, 16, "int8", "bf16", tokens=4096),
        # a short cached prefix read back for the prompt that continues it
        _cache("read_prefix", "read", 1, 1001, 8, 128, 16, 16, "int8", "bf16"),
        # cached prefixes of a batch
        _cache("read_batch", "read", 16, 8192, 8, 128, 128, 64, "e4m3", "fp16"),
        # one request's decode step: latency
        _cache("attend_one", "attend", 1, 777, 8, 128, 16, 16, "int8", "bf16", q_heads=32, queries=1, softcap=0.0, weights=False),
        # the decode batch of the repository's benchmark, its cache in 8 bits
        _cache("attend_batch", "attend", 64, 8192, 8, 128, 128, 16, "e4m3", "bf16", q_heads=32, queries=1, softcap=0.0, weights=False),
        # few long contexts, capped scores
        _cache("attend_long", "attend", 3, 131071, 8, 128, 64, 32, "int8", "fp16", q_heads=64, queries=1, softcap=50.0, weights=False),
        # four drafted tokens a request checked at once, attention weights accumulated for the eviction
        _cache("attend_verify", "attend", 24, 6000, 4, 128, 64, 64, "int8", "bf16", q_heads=32, queries=4, softcap=0.0, weights=True),
        # one long request cut to a budget
        _cache("evict_one", "evict", 1, 100003, 8, 128, 64, 16, "e4m3", "bf16", budget=16384, recent=1024),
        # a batch cut to a budget, some of it shorter than that
        _cache("evict_batch", "evict", 48, 8192, 8, 128, 128, 16, "e4m3", "bf16", budget=2048, recent=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "write", "read", "attend", "attend", "evict"])
    dtype = rng.choice(["bf16", "fp16"])
    head_dim = rng.choice([64, 128, 128, 256])
    block_size = rng.choice([16, 32, 64, 128])
    group = rng.choice([g for g in (16, 32, 64, 128) if block_size % g == 0])
    cache = rng.choice(["int8", "e4m3"])
    kv_heads = rng.choice([1, 2, 4, 8])
    if op == "rotary":
        d = rng.choice([64, 80, 128, 256])
        rot = rng.choice([d, d, d // 2 // 2 * 2])
        c = _rotary("", _log(rng, 1, 12000), kv_heads * rng.choice([1, 2, 4]), kv_heads, d, rot, rng.choice([1, 2, 3]), rng.random() < 0.5, rng.random() < 0.5, dtype)
    elif op == "write":
        # codes of 8 bits come back as they are; integer codes as the values they stand for
        if rng.random() < 0.5:
            c = _cache("", "write", _log(rng, 1, 128), _log(rng, 1, 4000), kv_heads, head_dim, block_size, group, "e4m3", dtype, tokens=1)
        else:
            c = _cache("", "write", _log(rng, 1, 16), _log(rng, 1, 800), kv_heads, head_dim, block_size, group, cache, dtype, tokens=_log(rng, 1, 3000))
    elif op == "read":
        c = _cache("", "read", _log(rng, 1, 24), _log(rng, 1, 4000), kv_heads, head_dim, block_size, group, cache, dtype)
    elif op == "attend":
        seqs = _log(rng, 1, 64)
        most = 200000 * 64 // (seqs * kv_heads * (head_dim // 64))
        c = _cache("", "attend", seqs, _log(rng, 1, min(100000, most)), kv_heads, head_dim, block_size, group, cache, dtype,
                   q_heads=kv_heads * rng.choice([1, 4, 5, 8, 16]), queries=rng.choice([1, 1, 1, 2, 3]), softcap=rng.choice([0.0, 0.0, 30.0]),
                   weights=rng.random() < 0.3)
    else:
        seqs = _log(rng, 1, 32)
        context = _log(rng, 64, min(100000, 250000 // seqs))
        budget = max(1, int(context * rng.uniform(0.1, 0.9)))
        c = _cache("", "evict", seqs, context, kv_heads, head_dim, block_size, group, "e4m3", dtype, budget=budget, recent=budget // rng.choice([2, 4, 8]))
    del c["name"]
    return c


# ----------------------------------------------------------------------------- inputs
def _ragged(n, most, seed):
    """n lengths spread evenly up to `most` (the longest has it), in an order of the seed's."""
    g = torch.Generator().manual_seed(seed)
    return torch.tensor([max(1, -(-(i + 1) * most // n)) for i in range(n)])[torch.randperm(n, generator=g)]


def _old_lens(c, seed):
    """Rows that each sequence has in the cache before a write: every fourth sequence of a prompt's batch continues a prefix."""
    if c["tokens"] == 1:
        return _ragged(c["seqs"], c["context"], seed)
    return torch.tensor([c["context"] if i % 4 == 1 else 0 for i in range(c["seqs"])])


def _new_lens(c, seed):
    return torch.ones(c["seqs"], dtype=torch.int64) if c["tokens"] == 1 else _ragged(c["seqs"], c["tokens"], seed + 1)


def _cum(lens):
    return torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)


def _quantised(shape, group, codes, gen):
    """A pool of rows N(0,1) times a size of its own for each head, in codes and scales, made page block by page block."""
    nb, heads, rows, d = shape
    cache = torch.empty(shape, dtype=codes, device=DEV)
    scale = torch.empty(nb, heads, rows // group, dtype=torch.float32, device=DEV)
    size = torch.exp(0.5 * torch.randn(1, heads, 1, 1, device=DEV, generator=gen))
    step = max(1, (1 << 27) // (heads * rows * d))
    for b in range(0, nb, step):
        n = min(step, nb - b)
        x = (torch.randn(n, heads, rows, d, device=DEV, generator=gen) * size).view(n, heads, rows // group, group * d)
        s = x.abs().amax(-1) / QMAX[codes]
        y = x / s[..., None]
        cache[b:b + n] = (y.round() if codes == torch.int8 else y).view(n, heads, rows, d).to(codes)
        scale[b:b + n] = s
    return cache, scale


def _paged(c, lens, seed, gen):
    P = c["block_size"]
    used = -(-lens // P)
    nb, width = int(used.sum()) + 3, int(used.max())
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed + 7)).to(torch.int32)
    tables = torch.zeros(c["seqs"], width, dtype=torch.int32)
    at = 0
    for s in range(c["seqs"]):
        tables[s, :int(used[s])] = perm[at:at + int(used[s])]
        at += int(used[s])
    shape = (nb, c["kv_heads"], P, c["head_dim"])
    k, ks = _quantised(shape, c["group"], CODES[c["cache"]], gen)
    v, vs = _quantised(shape, c["group"], CODES[c["cache"]], gen)
    return dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, block_tables=tables.to(DEV))


def _sections(c):
    half, axes = c["rot_dim"] // 2, c["axes"]
    return [half // axes + (1 if a >= axes - half % axes else 0) for a in range(axes)]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=c)
    if c["op"] == "rotary":
        T, dt = c["tokens"], TYPES[c["dtype"]]
        st["q"] = torch.randn(T, c["q_heads"], c["head_dim"], device=DEV, generator=gen).to(dt)
        st["k"] = torch.randn(T, c["kv_heads"], c["head_dim"], device=DEV, generator=gen).to(dt)
        t = torch.arange(T, device=DEV) + seed % 1000
        # frames of 24 x 32 patches: time, row and column of each patch
        grid = torch.stack([t, t % 768 // 32, t % 32] if c["axes"] == 3 else [t // 32, t % 32] if c["axes"] == 2 else [t], 1)
        st["positions"] = grid.to(torch.int32)
        i = torch.arange(c["rot_dim"] // 2, device=DEV, dtype=torch.float64)
        st["inv_freq"] = (10000.0 ** (-2.0 * i / c["rot_dim"])).to(torch.float32)
        st["sections"] = _sections(c)
        return st
    if c["op"] == "write":
        old, new = _old_lens(c, seed), _new_lens(c, seed)
        st.update(_paged(c, old + new, seed, gen))
        T = int(new.sum())
        size = torch.exp(0.5 * torch.randn(1, c["kv_heads"], 1, device=DEV, generator=gen))
        st["k"], st["v"] = ((torch.randn(T, c["kv_heads"], c["head_dim"], device=DEV, generator=gen) * size).to(TYPES[c["dtype"]]) for _ in range(2))
        st["old_lens"] = old.to(DEV, torch.int32)
        st["cu_new"] = None if c["tokens"] == 1 else _cum(new).to(DEV)
        st["cu_all"], st["total"] = _cum(old + new).to(DEV), int((old + new).sum())
        return st
    lens = _ragged(c["seqs"], c["context"], seed)
    st.update(_paged(c, lens, seed, gen))
    st["context_lens"] = lens.to(DEV, torch.int32)
    if c["op"] == "read":
        st["cu_all"], st["total"] = _cum(lens).to(DEV), int(lens.sum())
    width = st["block_tables"].shape[1] * c["block_size"]
    if c["op"] == "attend":
        shape = (c["seqs"], c["q_heads"], c["head_dim"]) if c["queries"] == 1 else (c["seqs"], c["queries"], c["q_heads"], c["head_dim"])
        st["q"] = torch.randn(shape, device=DEV, generator=gen).to(TYPES[c["dtype"]])
        st["weights"] = torch.zeros(c["seqs"], c["kv_heads"], width, device=DEV) if c["weights"] else None
    if c["op"] == "evict":
        # sums of attention weights: a few large, many small, some never attended to
        w = torch.rand(c["seqs"], c["kv_heads"], width, device=DEV, generator=gen)
        st["weights"] = torch.where(w < 0.1, torch.zeros_like(w), w ** 8)
        st["budget"], st["recent"] = c["budget"], c["recent"]
    return st


# ----------------------------------------------------------------------------- one pass
def _modules():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton-ascend-kernels_b200", "attention")
    if at not in sys.path:
        sys.path.insert(0, at)
    import kv8_cache
    import paged_attention_kv8
    import rotary_nd
    return rotary_nd, kv8_cache, paged_attention_kv8


def run(state):
    c, s = state["case"], state
    if own:
        rotary_nd, kv8, att = _modules()
        if c["op"] == "rotary":
            return rotary_nd.rotary_nd(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], interleaved=c["interleaved"], inverse=c["inverse"])
        cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_tables"])
        if c["op"] == "write":
            kv8.kv8_cache_write(s["k"], s["v"], *cache, s["old_lens"], s["cu_new"])
            if c["cache"] == "int8":
                return kv8.kv8_cache_read(*cache, s["cu_all"], s["total"], dtype=s["k"].dtype)
            return cache[:4]
        if c["op"] == "read":
            return kv8.kv8_cache_read(*cache, s["cu_all"], s["total"], dtype=TYPES[c["dtype"]])
        if c["op"] == "attend":
            out, lse = att.paged_attention_kv8(s["q"], *cache, s["context_lens"], softcap=c["softcap"], weights=s["weights"], return_lse=True)
            return out, lse, s["weights"]
        kept, lens = kv8.kv8_cache_evict(*cache, s["context_lens"], s["weights"], s["budget"], s["recent"])
        return kept, lens, s["weights"], cache[:4]
    if c["op"] == "rotary":
        return _plain_rotary(s, c)
    if c["op"] == "write":
        _plain_write(s, c, "k")
        _plain_write(s, c, "v")
        if c["cache"] == "int8":
            return _plain_read(s, c, "k"), _plain_read(s, c, "v")
        return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if c["op"] == "read":
        return _plain_read(s, c, "k"), _plain_read(s, c, "v")
    if c["op"] == "attend":
        return _plain_attend(s, c)
    return _plain_evict(s, c)


def _bytes(cache):
    return cache.view(torch.int8)


def _encode(x, codes):
    return x.round().to(codes) if codes == torch.int8 else x.to(codes)


def _plain_rotary(s, c):
    half, rot = c["rot_dim"] // 2, c["rot_dim"]
    sections = torch.tensor(s["sections"], device=DEV)
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=DEV), sections, output_size=half)
    angle = s["positions"][:, axis].float() * s["inv_freq"]
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    if c["inverse"]:
        sin = -sin

    def turn(x):
        y = x.float()
        a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if c["interleaved"] else (y[..., :half], y[..., half:rot])
        p, q = a * cos - b * sin, a * sin + b * cos
        z = torch.stack([p, q], -1).flatten(-2) if c["interleaved"] else torch.cat([p, q], -1)
        return torch.cat([z, y[..., rot:]], -1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _rows(s, c, cu, start, total):
    """(sequence, page, row in it) of each row that cu lists, the first of a sequence at its `start`."""
    t = torch.arange(total, device=DEV)
    seq = torch.searchsorted(cu[1:].long(), t, right=True)
    pos = t - cu.long()[seq] + (0 if start is None else start.long()[seq])
    return pos, s["block_tables"].long()[seq, pos // c["block_size"]], pos % c["block_size"]


def _plain_write(s, c, which):
    """Codes of the new rows under their group's scale, which grows where they need it; a group that grows has its earlier rows in the new scale too."""
    x, cache, scale = s[which].float(), s[which + "_cache"], s[which + "_scale"]
    g, P, codes, old = c["group"], c["block_size"], cache.dtype, s["old_lens"].long()
    T, heads = x.shape[:2]
    cu = torch.arange(T + 1, device=DEV) if s["cu_new"] is None else s["cu_new"].long()
    pos, page, row = _rows(s, c, cu, old, T)
    ng = P // g
    group = page * ng + row // g
    amax = torch.zeros(scale.shape[0] * ng, heads, device=DEV).scatter_reduce_(0, group[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    want = torch.where(amax < TINY, torch.zeros_like(amax), amax * (1.0 / QMAX[codes]))
    touched = torch.zeros(amax.shape[0], 1, dtype=torch.bool, device=DEV)
    touched[group] = True
    first = torch.zeros(amax.shape[0], device=DEV).index_add_(0, group, (pos % g == 0).float())[:, None] > 0
    before = scale.permute(0, 2, 1).reshape(-1, heads)
    after = torch.where(touched, torch.where(first, want, torch.maximum(before, want)), before)
    # the open group of each sequence
    at = s["block_tables"].long().gather(1, (old // P).clamp(max=s["block_tables"].shape[1] - 1)[:, None])[:, 0]
    rows = (old % P // g * g)[:, None] + torch.arange(g, device=DEV)
    gid = at * ng + old % P // g
    grown = (before[gid] < after[gid]) & (cu[1:] > cu[:-1])[:, None] & (old % g > 0)[:, None]
    ratio = torch.where(grown, before[gid] / after[gid], torch.ones_like(after[gid]))
    held = _bytes(cache)[at[:, None], :, rows].view(codes)
    mine = (torch.arange(g, device=DEV) < (old % g)[:, None])[:, :, None] & grown[:, None]
    again = _encode(held.float() * ratio[:, None, :, None], codes)
    _bytes(cache)[at[:, None], :, rows] = torch.where(mine[..., None], _bytes(again), _bytes(held))
    inv = torch.where(after > 0, 1.0 / after, torch.zeros_like(after))[group]
    _bytes(cache)[page, :, row] = _bytes(_encode(x * inv[..., None], codes))
    scale.copy_(after.view(scale.shape[0], ng, heads).permute(0, 2, 1))


def _plain_read(s, c, which):
    cache, scale = s[which + "_cache"], s[which + "_scale"]
    _, page, row = _rows(s, c, s["cu_all"], None, s["total"])
    x = _bytes(cache)[page, :, row].view(cache.dtype).float() * scale[page, :, row // c["group"]][..., None]
    return x.to(TYPES[c["dtype"]])


def _plain_attend(s, c):
    B, H, Hkv, D, L, Q = c["seqs"], c["q_heads"], c["kv_heads"], c["head_dim"], c["context"], c["queries"]
    pos = torch.arange(L, device=DEV)
    page, row = s["block_tables"].long()[:, pos // c["block_size"]], pos % c["block_size"]
    q = s["q"].float().view(B, Q, Hkv, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B * Hkv, -1, D)

    def values(which):
        cache, scale = s[which + "_cache"], s[which + "_scale"]
        x = _bytes(cache)[page, :, row].view(cache.dtype).float() * scale[page, :, row // c["group"]][..., None]
        return x.permute(0, 2, 1, 3).reshape(B * Hkv, L, D)

    z = torch.bmm(q, values("k").transpose(1, 2)) / math.sqrt(D)
    if c["softcap"]:
        z = c["softcap"] * torch.tanh(z / c["softcap"])
    limit = s["context_lens"].long()[:, None] - Q + 1 + torch.arange(Q, device=DEV)
    seen = (pos < limit[..., None])[:, None, :, None].expand(B, Hkv, Q, H // Hkv, L).reshape(z.shape)
    z = torch.where(seen, z, torch.full_like(z, -math.inf))
    top = z.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).view(B, Hkv, Q, H // Hkv).permute(0, 2, 1, 3).reshape(B, Q, H)
    out = torch.bmm(p, values("v")).view(B, Hkv, Q, H // Hkv, D).permute(0, 2, 1, 3, 4).reshape(B, Q, H, D).to(s["q"].dtype)
    if s["weights"] is not None:
        s["weights"][:, :, :L] += p.view(B, Hkv, -1, L).sum(2)
    return (out, lse, s["weights"]) if Q > 1 else (out[:, 0], lse[:, 0], s["weights"])


def _plain_evict(s, c):
    w, n = s["weights"], s["context_lens"].long()[:, None, None]
    B, Hkv, W = w.shape
    P, g, budget, recent = c["block_size"], c["group"], min(c["budget"], W), c["recent"]
    pos = torch.arange(W, device=DEV).expand(B, Hkv, W)
    rank = torch.where(pos >= n, 2, torch.where(pos >= n - recent, 0, 1))
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(rank.gather(-1, order), dim=-1, stable=True).indices)
    slot = torch.arange(c["budget"], device=DEV)
    lens = torch.minimum(s["context_lens"].long(), torch.tensor(c["budget"], device=DEV))
    real = (slot < lens[:, None])[:, None].expand(B, Hkv, -1)
    kept = torch.cat([order[..., :budget], torch.zeros(B, Hkv, c["budget"] - budget, dtype=order.dtype, device=DEV)], -1)
    kept = torch.sort(torch.where(real, kept, torch.full_like(kept, 1 << 40)), -1).values
    kept = torch.where(real, kept, torch.full_like(kept, -1))
    src = kept.clamp(min=0)
    b, h = torch.arange(B, device=DEV)[:, None, None], torch.arange(Hkv, device=DEV)[:, None]
    table = s["block_tables"].long()
    at = real[:, :, :W]
    spage, srow = table[b, src // P], src % P
    to = slot[:W].expand(B, Hkv, -1)
    dpage, drow = table[b, to // P], to % P
    pad = (-c["budget"]) % g
    for which in ("k", "v"):
        cache, scale = s[which + "_cache"], s[which + "_scale"]
        held = _bytes(cache)[spage, h, srow].view(cache.dtype)
        was = torch.where(real, scale[spage, h, srow // g], torch.zeros((), device=DEV))
        most = torch.nn.functional.pad(was, (0, pad)).view(B, Hkv, -1, g).amax(-1)
        now = most.repeat_interleave(g, -1)[..., :c["budget"]]
        ratio = torch.where(was < now, was / now, torch.ones_like(now))
        again = _encode(held.float() * ratio[..., None], cache.dtype)
        bb, hh = b.expand(B, Hkv, at.shape[-1])[at], h.expand(B, Hkv, at.shape[-1])[at]
        _bytes(cache)[dpage[at], hh, drow[at]] = _bytes(again)[:, :, :W][at]
        scale[dpage[at], hh, drow[at] // g] = now[:, :, :W][at]
    moved = torch.where(real, w.gather(-1, src.clamp(max=W - 1)), torch.zeros((), device=DEV))[..., :W]
    moved = torch.nn.functional.pad(moved, (0, W - moved.shape[-1]))
    s["weights"].copy_(torch.where(pos < n, moved, w))
    return kept.to(torch.int32), lens.to(torch.int32), s["weights"], (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])


# ----------------------------------------------------------------------------- what one pass cannot do without
def _lens(c):
    return [max(1, -(-(i + 1) * c["context"] // c["seqs"])) for i in range(c["seqs"])]


def work(case):
    c = case
    if c["op"] == "rotary":
        n = c["tokens"] * (c["q_heads"] + c["kv_heads"])
        return dict(bytes=2 * 2 * n * c["head_dim"] + 4 * c["tokens"] * c["axes"], flops=3 * n * c["rot_dim"])
    D, Hkv, g = c["head_dim"], c["kv_heads"], c["group"]
    row = 2 * Hkv * D  # a token's codes, K and V
    tag = 2 * Hkv * 4 / g  # its share of the scales
    if c["op"] == "write":
        old = sum(int(x) for x in _old_lens(c, 0))
        new = sum(int(x) for x in _new_lens(c, 0))
        n = 3 * row * new + 2 * tag * new
        if c["cache"] == "int8":
            n += (old + new) * (row + tag + 2 * row)
        return dict(bytes=n, flops=2 * row * new)
    keys = sum(_lens(c))
    if c["op"] == "read":
        return dict(bytes=keys * (3 * row + tag), flops=keys * row)
    if c["op"] == "attend":
        rows = c["q_heads"] * c["queries"]
        return dict(bytes=keys * (row + tag) + c["seqs"] * rows * (4 * D + 4) + (8 * keys * Hkv if c["weights"] else 0), flops=4 * keys * rows * D)
    kept = sum(min(n, c["budget"]) for n in _lens(c))
    cut = sum(min(n, c["budget"]) for n in _lens(c) if n > c["budget"])
    return dict(bytes=4 * Hkv * (keys + 2 * kept) + 2 * cut * (row + tag), flops=2 * cut * row)


# ----------------------------------------------------------------------------- 64 bits
def _e4m3(x):
    """x rounded to the nearest value of e4m3 (three bits of mantissa, exponents from -6, largest 448), ties to even."""
    _, e = torch.frexp(x)
    q = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / q) * q).clamp(-448, 448)


def _near(x, codes):
    return torch.round(x).clamp(-127, 127) if codes == torch.int8 else _e4m3(x)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f = torch.float64
    if c["op"] == "rotary":
        axis = [a for a, n in enumerate(s["sections"]) for _ in range(n)]
        z = torch.polar(torch.ones((), dtype=f, device=DEV), s["positions"].to(f)[:, axis] * s["inv_freq"].to(f) * (-1 if c["inverse"] else 1))[:, None]

        def spin(x):
            y, r = x.to(f), c["rot_dim"]
            pairs = y[..., :r].unflatten(-1, (r // 2, 2)) if c["interleaved"] else y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
            w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
            y[..., :r] = (w if c["interleaved"] else w.transpose(-1, -2)).flatten(-2)
            return y

        return spin(s["q"]), spin(s["k"])
    table, P, g, D, Hkv = s["block_tables"].long(), c["block_size"], c["group"], c["head_dim"], c["kv_heads"]
    codes = CODES[c["cache"]]

    def sequence(which, b, n, whole=None):
        """Codes [n, heads, D] and scales [n, heads] of a sequence's first n rows."""
        cache, scale = (s[which + "_cache"], s[which + "_scale"]) if whole is None else whole
        pages = table[b, :-(-n // P)]
        x = _bytes(cache)[pages].view(cache.dtype).to(f) if whole is None else cache[pages]
        return x.transpose(1, 2).flatten(0, 1)[:n], scale[pages].to(f).transpose(1, 2).flatten(0, 1).repeat_interleave(g, 0)[:n]

    if c["op"] == "read":
        got = {w: [x * t[..., None] for b in range(c["seqs"]) for x, t in [sequence(w, b, int(s["context_lens"][b]))]] for w in "kv"}
        return torch.cat(got["k"]), torch.cat(got["v"])
    if c["op"] == "attend":
        outs, lses, ws = [], [], []
        Q, G = c["queries"], c["q_heads"] // Hkv
        for b in range(c["seqs"]):
            n = int(s["context_lens"][b])
            (k, ks), (v, vs) = sequence("k", b, n), sequence("v", b, n)
            q = s["q"][b].to(f).view(Q, Hkv, G, D)
            z = torch.einsum("qhgd,nhd->qhgn", q, k * ks[..., None]) / D ** 0.5
            if c["softcap"]:
                z = torch.tanh(z / c["softcap"]) * c["softcap"]
            late = torch.arange(n, device=DEV) > (n - Q + torch.arange(Q, device=DEV))[:, None]
            z.masked_fill_(late[:, None, None], -math.inf)
            l = torch.logsumexp(z, -1)
            p = torch.exp(z - l.clamp(min=-1e300)[..., None])
            outs.append(torch.einsum("qhgn,nhd->qhgd", p, v * vs[..., None]).reshape(Q, -1, D))
            lses.append(l.reshape(Q, -1))
            if s["weights"] is not None:
                w = torch.zeros(Hkv, s["weights"].shape[2], dtype=f, device=DEV)
                w[:, :n] = p.sum((0, 2))
                ws.append(w)
        out, lse = torch.stack(outs), torch.stack(lses)
        return (out, lse, torch.stack(ws) if ws else None) if Q > 1 else (out[:, 0], lse[:, 0], torch.stack(ws) if ws else None)
    pool = {w: (_bytes(s[w + "_cache"]).view(codes).to(f), s[w + "_scale"].to(f)) for w in "kv"}
    if c["op"] == "write":
        old = s["old_lens"].tolist()
        cu = list(range(len(old) + 1)) if s["cu_new"] is None else s["cu_new"].tolist()
        for w in "kv":
            cache, scale = pool[w]
            for b, start in enumerate(old):
                x, end = s[w][cu[b]:cu[b + 1]].to(f), start + cu[b + 1] - cu[b]
                lead = start % g
                have, t = sequence(w, b, start, pool[w])
                have, t = have[start - lead:], t[start - lead:]
                n = -(-(end - (start - lead)) // g)
                y = torch.zeros(n * g, Hkv, D, dtype=f, device=DEV)
                y[lead:lead + len(x)] = x
                want = y.view(n, g, Hkv, D).abs().amax((1, 3)) / QMAX[codes]
                if lead:
                    want[0] = torch.maximum(want[0], t[0])
                y = _near(y.view(n, g, Hkv, D) / want[:, None, :, None].clamp(min=1e-300), codes).view(n * g, Hkv, D)
                if lead:
                    y[:lead] = _near(have * (t[0] / want[0])[:, None], codes)
                p = torch.arange(start - lead, end, device=DEV)
                cache[table[b, p // P], :, p % P] = y[:len(p)]
                scale[table[b, p // P], :, p % P // g] = want.repeat_interleave(g, 0)[:len(p)]
        if c["cache"] == "int8":
            got = {w: [x * t[..., None] for b in range(c["seqs"]) for x, t in [sequence(w, b, old[b] + cu[b + 1] - cu[b], pool[w])]] for w in "kv"}
            return torch.cat(got["k"]), torch.cat(got["v"])
        return pool["k"][0], pool["v"][0], pool["k"][1], pool["v"][1]
    weights = s["weights"].to(f)
    for b, n in enumerate(s["context_lens"].tolist()):
        m = min(n, c["budget"])
        first = n - min(c["recent"], n)
        if n > m:
            by = torch.sort(weights[b, :, :first], dim=-1, descending=True, stable=True).indices[:, :m - c["recent"]]
            keep = torch.cat([torch.sort(by, dim=-1).values, torch.arange(first, n, device=DEV).expand(Hkv, -1)], -1)
        else:
            keep = torch.arange(n, device=DEV).expand(Hkv, -1)
        to = torch.arange(m, device=DEV)
        heads = torch.arange(Hkv, device=DEV)[:, None]
        for w in "kv":
            cache, scale = pool[w]
            page = table[b, keep // P]
            x, t = cache[page, heads, keep % P], scale[page, heads, keep % P // g]
            n_g = -(-m // g)
            u = torch.zeros(Hkv, n_g * g, dtype=f, device=DEV)
            u[:, :m] = t
            u = u.view(Hkv, n_g, g).amax(-1)
            big = u.repeat_interleave(g, -1)[:, :m]
            cache[table[b, to // P], heads, to % P] = _near(x * (t / big)[..., None], codes)
            scale[table[b, to // P], heads, to % P // g] = big
        moved = weights[b].gather(-1, keep)
        weights[b, :, :n] = 0
        weights[b, :, :m] = moved
    return None, None, weights, (pool["k"][0], pool["v"][0], pool["k"][1], pool["v"][1])
