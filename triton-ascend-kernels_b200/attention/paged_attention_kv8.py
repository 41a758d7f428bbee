"""Paged attention over the 8-bit KV cache of ``kv8_cache`` on B200.

An addition without a counterpart in suluner/triton-ascend-kernels: the
attention of a decode step (or of a few drafted tokens per request) whose K and
V are held in 8 bits with a scale for each page, head and group of rows.
"""

import math
import struct

import _tak_b200 as _t
from kv8_cache import _lens, describe

_KEEP = 256 << 20  # bytes of scratch that a stream keeps at most
_MIN_CAP = 2.0 ** -126  # fp32's smallest normal number: its reciprocal is finite
_S3, _S4 = struct.Struct("=3q").pack, struct.Struct("=4q").pack


def paged_attention_kv8(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, *, softcap=0.0,
                        weights=None, return_lse=False):
    """Attention of the newest tokens of each sequence over its cached rows.
    Scores are q . k / sqrt(head_dim).

    Args:
        q: [num_seqs, num_q_heads, head_dim], or [num_seqs, num_queries,
            num_q_heads, head_dim] for several new tokens per sequence
        k_cache, v_cache, k_scale, v_scale: the cache (see kv8_cache)
        block_tables: [num_seqs, max_blocks] int32 page ids
        context_lens: [num_seqs] int32 cached rows, the new tokens' among
            them: query i of num_queries sees the first context_lens[s] -
            num_queries + 1 + i
        softcap: > 0 caps the scaled scores: z -> softcap * tanh(z / softcap);
            0, and all above 2^126, cap nothing
        weights: [num_seqs, num_kv_heads, max_rows] float32; each key's
            attention weight, summed over the query rows and heads that share
            its KV head, is added to it (what kv8_cache_evict ranks by)
        return_lse: also return the natural log of each row's softmax
            denominator, float32, q's shape without head_dim

    A row that sees no key gives zeros (lse -inf).
    """
    desc, _bt, (index, hkv, d, seqs) = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    shape = q.shape
    assert len(shape) in (3, 4), "q must be [num_seqs, num_q_heads, head_dim] or [num_seqs, num_queries, ...]"
    assert q.get_device() == index and (weights is None or weights.get_device() == index), \
        "q and weights must be on the cache's CUDA device"
    B, H, D = shape[0], shape[-2], shape[-1]
    Lq = shape[1] if len(shape) == 4 else 1
    assert B == seqs, "block_tables must have a row per sequence"
    assert D == d, f"head_dim of q ({D}) and of the cache ({d}) differ"
    assert H % hkv == 0, f"num_q_heads ({H}) must be divisible by num_kv_heads ({hkv})"
    assert softcap == 0.0 or softcap >= _MIN_CAP, "softcap must be 0 (none) or at least 2^-126"
    cl = _lens(context_lens, index, seqs, "context_lens")
    st = q.stride()
    if len(st) == 3:
        st = (st[0], 0, st[1], st[2])
    wp = wst = None
    width = 0
    if weights is not None:
        ws = weights.shape
        assert len(ws) == 3 and ws[0] == B and ws[1] == hkv and weights.dtype is _t.torch.float32, \
            "weights must be float32 [num_seqs, num_kv_heads, max_rows]"
        width = ws[2]
        wp, wst = weights.data_ptr(), _S3(*weights.stride())
    out = _t.like(q)
    lse = _t.torch.empty_strided(shape[:-1], (H, 1) if len(shape) == 3 else (Lq * H, H, 1), dtype=_t.torch.float32,
                                 device=q.device) if return_lse else None
    L = _t.lib()
    stream = _t.raw_stream(index)
    code = _t.dtype_code(q)
    if _t.capturing():
        # a graph's scratch is its own: the stream's may be replaced before a replay, or be
        # in use beside it
        scratch = _t.torch.empty(L.tak_kv8_attention_workspace_size(desc, H, Lq, width, code),
                                 dtype=_t.torch.uint8, device=q.device)
    else:
        scratch = _t.workspace_of(index, stream)
    while True:
        rc = L.tak_kv8_attention(
            desc, q.data_ptr(), _S4(*st), cl.data_ptr(), out.data_ptr(), _S4(Lq * H * D, H * D, D, 1),
            None if lse is None else lse.data_ptr(), wp, wst, width, H, Lq, 1.0 / math.sqrt(D), softcap, code,
            scratch.data_ptr(), scratch.numel(), stream)
        if rc != 4:  # 4: the workspace is too small; nothing was launched
            break
        need = L.tak_kv8_attention_workspace_size(desc, H, Lq, width, code)
        # the scores of a long call with weights go back to the allocator after it
        scratch = _t.workspace_of(index, stream, need) if need <= _KEEP else \
            _t.torch.empty(need, dtype=_t.torch.uint8, device=q.device)
    if rc:
        _t.check(rc)
    return (out, lse) if return_lse else out
