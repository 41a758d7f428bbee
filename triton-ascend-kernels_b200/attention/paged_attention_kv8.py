"""Paged attention over the 8-bit KV cache of ``kv8_cache`` on B200.

An addition without a counterpart in suluner/triton-ascend-kernels: the
attention of a decode step (or of a few drafted tokens per request) whose K and
V are held in 8 bits with a scale for each page, head and group of rows.
"""

import math

import _tak_b200 as _t
from kv8_cache import describe


def paged_attention_kv8(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, *, softcap=0.0,
                        weights=None, return_lse=False):
    """Attention of the newest tokens of each sequence over its cached rows.

    Args:
        q: [num_seqs, num_q_heads, head_dim], or [num_seqs, num_queries,
            num_q_heads, head_dim] for several new tokens per sequence
        k_cache, v_cache, k_scale, v_scale: the cache (see kv8_cache)
        block_tables: [num_seqs, max_blocks] int32 page ids
        context_lens: [num_seqs] int32 cached rows, the new tokens' among
            them: query i of num_queries sees the first context_lens[s] -
            num_queries + 1 + i
        softcap: > 0 caps the scaled scores: z -> softcap * tanh(z / softcap)
        weights: [num_seqs, num_kv_heads, max_rows] float32; each key's
            attention weight, summed over the query rows and heads that share
            its KV head, is added to it (what kv8_cache_evict ranks by)
        return_lse: also return the natural log of each row's softmax
            denominator, float32, q's shape without head_dim

    A row that sees no key gives zeros (lse -inf).
    """
    _t.require_cuda(q)
    d, bt = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    assert q.dim() in (3, 4), "q must be [num_seqs, num_q_heads, head_dim] or [num_seqs, num_queries, ...]"
    q4 = q if q.dim() == 4 else q.unsqueeze(1)
    B, Lq, H, D = q4.shape
    hkv = k_cache.shape[1]
    assert B == bt.shape[0], "block_tables must have a row per sequence"
    assert D == k_cache.shape[3], f"head_dim of q ({D}) and of the cache ({k_cache.shape[3]}) differ"
    assert H % hkv == 0, f"num_q_heads ({H}) must be divisible by num_kv_heads ({hkv})"
    assert softcap >= 0.0, "softcap must be >= 0"
    cl = _t.as_i32(context_lens, q.device)
    assert cl.dim() == 1 and cl.shape[0] == B, "context_lens must be [num_seqs]"
    cl = cl.contiguous()
    width = 0
    if weights is not None:
        _t.require_cuda(weights)
        assert weights.dim() == 3 and weights.shape[:2] == (B, hkv) and weights.dtype == _t.torch.float32, \
            "weights must be float32 [num_seqs, num_kv_heads, max_rows]"
        width = weights.shape[2]
    out = q.new_empty(q.shape)
    out4 = out if q.dim() == 4 else out.unsqueeze(1)
    lse = q.new_empty(q.shape[:-1], dtype=_t.torch.float32) if return_lse else None
    L = _t.lib()
    st = _t.stream_of(q)
    code = _t.dtype_code(q)
    need = L.tak_kv8_attention_workspace_size(d, H, Lq, width, code)
    ws = _t.workspace(q.device, st, max(need, 0))
    _t.check(L.tak_kv8_attention(
        d, _t.ptr(q4), _t.strides(q4), _t.ptr(cl), _t.ptr(out4), _t.strides(out4), _t.ptr(lse), _t.ptr(weights),
        None if weights is None else _t.strides(weights), width, H, Lq, 1.0 / math.sqrt(D), float(softcap), code,
        _t.ptr(ws), ws.numel(), st))
    return (out, lse) if return_lse else out
