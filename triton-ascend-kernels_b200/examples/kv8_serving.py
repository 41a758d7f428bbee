"""A serving loop over the 8-bit paged KV cache, on random projections.

    python triton-ascend-kernels_b200/examples/kv8_serving.py

Prompts of images and text (three position axes) go through the rotary
positions, the varlen prefill and the cache's write; decode steps append one
token a request, attend over the cache and accumulate attention weights; when
the contexts pass a limit, each head keeps its heaviest and its most recent
rows; at the end one request gets another prompt, whose attention reads the
cached prefix back as 16-bit rows.  Beside it a 16-bit cache takes the same
rows, to show what the 8 bits cost.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "attention"))

from flash_attention_prefill import flash_attention_prefill  # noqa: E402
from kv8_cache import kv8_alloc, kv8_cache_evict, kv8_cache_read, kv8_cache_write  # noqa: E402
from paged_attention_decode import paged_attention_decode  # noqa: E402
from paged_attention_kv8 import paged_attention_kv8  # noqa: E402
from rotary_nd import rotary_nd  # noqa: E402


def positions_of(start, n, grid=(4, 6)):
    """(time, row, column) of n tokens from `start` on: frames of grid patches."""
    t = start + torch.arange(n)
    h, w = grid
    return torch.stack([t // (h * w), t % (h * w) // w, t % w], 1).to(torch.int32)


def main(prompts=(130, 700, 257, 64), steps=40, q_heads=32, kv_heads=8, head_dim=128, block=64, group=16,
         codes=torch.int8, limit=720, budget=256, recent=64, device="cuda", seed=0, verbose=True):
    g = torch.Generator(device=device).manual_seed(seed)
    B, dt = len(prompts), torch.bfloat16

    def rand(n, heads):
        return torch.randn(n, heads, head_dim, device=device, generator=g).to(dt)

    half = head_dim // 2
    inv_freq = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(device)
    sections = [half - 2 * (half // 3), half // 3, half // 3]

    # pages: every request gets a table for its longest context
    width = -(-(max(prompts) + steps) // block)
    tables = torch.randperm(B * width).view(B, width).to(device, torch.int32)
    cache = kv8_alloc(B * width, kv_heads, block, head_dim, group=group, dtype=codes, device=device)
    k16, v16 = (torch.zeros(B * width, kv_heads, block, head_dim, dtype=dt, device=device) for _ in range(2))
    weights = torch.zeros(B, kv_heads, width * block, device=device)

    # ---- prompts ----
    T = sum(prompts)
    cu = torch.tensor([0, *torch.tensor(prompts).cumsum(0)], dtype=torch.int32, device=device)
    pos = torch.cat([positions_of(0, n) for n in prompts]).to(device)
    q, k, v = rand(T, q_heads), rand(T, kv_heads), rand(T, kv_heads)
    rotary_nd(q, k, pos, inv_freq, sections, out=(q, k))
    flash_attention_prefill(q, k, v, cu, causal=True)
    start = torch.zeros(B, dtype=torch.int32, device=device)
    kv8_cache_write(k, v, *cache, tables, start, cu)
    ctx = (cu[1:] - cu[:-1]).clone()
    at = 0
    for s, n in enumerate(prompts):  # the 16-bit cache for comparison
        r = torch.arange(n, device=device)
        k16[tables[s, r // block].long(), :, r % block] = k[at:at + n]
        v16[tables[s, r // block].long(), :, r % block] = v[at:at + n]
        at += n

    # ---- decode ----
    seen = ctx.tolist()  # tokens so far: positions go on when rows are evicted
    worst, evictions, same = 0.0, 0, True
    for step in range(steps):
        q, k, v = rand(B, q_heads), rand(B, kv_heads), rand(B, kv_heads)
        pos = torch.cat([positions_of(n, 1) for n in seen]).to(device)
        rotary_nd(q, k, pos, inv_freq, sections, out=(q, k))
        kv8_cache_write(k, v, *cache, tables, ctx)
        seen = [n + 1 for n in seen]
        if same:
            page, row = tables.gather(1, (ctx // block).long()[:, None])[:, 0].long(), (ctx % block).long()
            k16[page, :, row], v16[page, :, row] = k, v
        ctx += 1
        out = paged_attention_kv8(q, *cache, tables, ctx, weights=weights)
        if same:
            ref = paged_attention_decode(q, k16, v16, tables, ctx, block, block)
            worst = max(worst, ((out.float() - ref.float()).norm() / ref.float().norm()).item())
        if int(ctx.max()) > limit:  # a server knows its contexts on the host
            kept, ctx = kv8_cache_evict(*cache, tables, ctx, weights, budget, recent)
            evictions += 1
            same = False

    # ---- another prompt for request 0, over its cached prefix ----
    n, more = int(ctx[0]), 100
    pk, pv = kv8_cache_read(*cache, tables[:1], torch.tensor([0, n], device=device, dtype=torch.int32), n, dtype=dt)
    q, k, v = rand(more, q_heads), rand(more, kv_heads), rand(more, kv_heads)
    rotary_nd(q, k, positions_of(seen[0], more).to(device), inv_freq, sections, out=(q, k))
    q = torch.cat([torch.zeros(n, q_heads, head_dim, dtype=dt, device=device), q])
    both = torch.tensor([0, n + more], dtype=torch.int32, device=device)
    answer = flash_attention_prefill(q, torch.cat([pk, k]), torch.cat([pv, v]), both, causal=True)[n:]

    if verbose:
        held = sum(t.numel() * t.element_size() for t in cache)
        print(f"{B} requests, {steps} steps, {evictions} evictions, contexts now {ctx.tolist()}")
        print(f"cache {held / 2**20:.1f} MiB against {2 * k16.numel() * 2 / 2**20:.1f} MiB in 16 bits; "
              f"largest relative difference of a step's output before the first eviction {worst:.4f}")
    return dict(worst=worst, evictions=evictions, contexts=ctx, weights=weights, answer=answer)


if __name__ == "__main__":
    main()
