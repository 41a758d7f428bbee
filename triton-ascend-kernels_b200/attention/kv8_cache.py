"""A paged KV cache held in 8 bits: allocation, write, read-back, eviction.

An addition without a counterpart in suluner/triton-ascend-kernels.  The cache
is four tensors: codes ``k_cache`` / ``v_cache`` [num_blocks, num_kv_heads,
block_size, head_dim] (torch.int8 or torch.float8_e4m3fn) and scales
``k_scale`` / ``v_scale`` [num_blocks, num_kv_heads, block_size / group]
(float32), one for each page, head and group of ``group`` consecutive rows.  An
element's value is code * scale.  ``paged_attention_kv8`` attends over it.
"""

import struct

import _tak_b200 as _t

_torch = _t.torch
_CODES = {_torch.int8: 0, _torch.float8_e4m3fn: 1}
_PACK = struct.Struct("=5q5q4q4q3q8q")  # struct tak_kv8_cache: every field 8 bytes


def kv8_alloc(num_blocks, num_kv_heads, block_size, head_dim, *, group=16, dtype=_torch.int8, device="cuda"):
    """Zeroed (k_cache, v_cache, k_scale, v_scale) of the given sizes."""
    assert dtype in _CODES, "dtype must be torch.int8 or torch.float8_e4m3fn"
    assert 1 <= group <= 256 and block_size % group == 0, \
        f"group ({group}) must divide block_size ({block_size}) and be at most 256"
    codes = [_torch.zeros(num_blocks, num_kv_heads, block_size, head_dim, dtype=_torch.int8,
                          device=device).view(dtype) for _ in range(2)]
    scales = [_torch.zeros(num_blocks, num_kv_heads, block_size // group, dtype=_torch.float32, device=device)
              for _ in range(2)]
    return (*codes, *scales)


def describe(k_cache, v_cache, k_scale, v_scale, block_tables):
    """The C ABI's description of a cache (struct tak_kv8_cache, as bytes) and
    the int32 block table that it points to."""
    _t.require_cuda(k_cache, v_cache, k_scale, v_scale)
    assert k_cache.dtype in _CODES, f"unsupported cache dtype {k_cache.dtype}: expected int8 or float8_e4m3fn"
    assert k_cache.dim() == 4 and v_cache.shape == k_cache.shape and v_cache.dtype == k_cache.dtype, \
        "k_cache and v_cache must be [num_blocks, num_kv_heads, block_size, head_dim] of one dtype"
    nb, hkv, rows, d = k_cache.shape
    assert k_scale.dim() == 3 and k_scale.shape[:2] == (nb, hkv) and v_scale.shape == k_scale.shape, \
        "k_scale and v_scale must be [num_blocks, num_kv_heads, block_size / group]"
    assert k_scale.dtype == _torch.float32 and v_scale.dtype == _torch.float32, "scales must be float32"
    ng = k_scale.shape[2]
    assert ng > 0 and rows % ng == 0, f"the number of scales ({ng}) must divide block_size ({rows})"
    bt = _t.as_i32(block_tables, k_cache.device)
    assert bt.dim() == 2, "block_tables must be [num_seqs, max_blocks]"
    return _PACK.pack(
        k_cache.data_ptr(), *k_cache.stride(), v_cache.data_ptr(), *v_cache.stride(),
        k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride(),
        bt.data_ptr(), *bt.stride(), nb, hkv, rows, d, rows // ng, bt.shape[0], bt.shape[1],
        _CODES[k_cache.dtype]), bt


def kv8_cache_write(k, v, k_cache, v_cache, k_scale, v_scale, block_tables, start_lens, cu_seqlens=None):
    """Write new rows into the cache, in place.

    Args:
        k, v: [total_tokens, num_kv_heads, head_dim] fp16, bf16 or fp32
        k_cache, v_cache, k_scale, v_scale: the cache
        block_tables: [num_seqs, max_blocks] int32 page ids
        start_lens: [num_seqs] int32 rows that each sequence already holds:
            its new rows go to positions start_lens[s] and on
        cu_seqlens: [num_seqs + 1] int32 row ranges of the sequences in k / v;
            None = one row per sequence (a decode step)

    A group's scale is its largest magnitude / 127 (int8) or / 448 (e4m3).
    Appending to a group that holds rows keeps the larger of the two scales;
    rows held under a smaller one are rounded again into it.
    """
    _t.require_cuda(k, v)
    d, bt = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    assert k.dim() == 3 and v.shape == k.shape and v.dtype == k.dtype, "K and V must have the same shape and dtype"
    assert k.shape[1] == k_cache.shape[1] and k.shape[2] == k_cache.shape[3], \
        "k / v must be [total_tokens, num_kv_heads, head_dim] of the cache"
    start = _t.as_i32(start_lens, k.device)
    assert start.dim() == 1 and start.shape[0] == bt.shape[0], "start_lens must be [num_seqs]"
    cu = None if cu_seqlens is None else _t.as_i32(cu_seqlens, k.device)
    assert cu is None or (cu.dim() == 1 and cu.shape[0] == bt.shape[0] + 1), "cu_seqlens must be [num_seqs + 1]"
    assert cu is not None or k.shape[0] == bt.shape[0], "without cu_seqlens k / v hold one row per sequence"
    start = start.contiguous()
    cu = None if cu is None else cu.contiguous()
    _t.check(_t.lib().tak_kv8_write(d, _t.ptr(k), _t.strides(k), _t.ptr(v), _t.strides(v), _t.ptr(start), _t.ptr(cu),
                                    k.shape[0], _t.dtype_code(k), _t.stream_of(k)))


def kv8_cache_read(k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens, total_tokens, *,
                   start_lens=None, dtype=_torch.bfloat16):
    """Read rows back as fp16, bf16 or fp32: (k, v) [total_tokens,
    num_kv_heads, head_dim], rows cu_seqlens[s] and on holding positions
    start_lens[s] (None: 0) and on of sequence s.  Rows outside every sequence
    are zeros."""
    d, bt = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    dev = k_cache.device
    cu = _t.as_i32(cu_seqlens, dev).contiguous()
    assert cu.dim() == 1 and cu.shape[0] == bt.shape[0] + 1, "cu_seqlens must be [num_seqs + 1]"
    start = None if start_lens is None else _t.as_i32(start_lens, dev).contiguous()
    assert start is None or (start.dim() == 1 and start.shape[0] == bt.shape[0]), "start_lens must be [num_seqs]"
    k = _torch.empty((int(total_tokens), k_cache.shape[1], k_cache.shape[3]), dtype=dtype, device=dev)
    v = _torch.empty_like(k)
    _t.check(_t.lib().tak_kv8_read(d, _t.ptr(cu), _t.ptr(start), k.shape[0], _t.ptr(k), _t.strides(k), _t.ptr(v),
                                   _t.strides(v), _t.dtype_code(k), _t.stream_of(k)))
    return k, v


def kv8_cache_evict(k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, weights, budget, recent):
    """Cut every sequence to at most `budget` rows per KV head, in place.

    Args:
        context_lens: [num_seqs] int32 rows that each sequence holds
        weights: [num_seqs, num_kv_heads, max_rows] float32 accumulated
            attention weights (paged_attention_kv8's `weights`)
        budget: rows that stay
        recent: the last `recent` rows stay whatever their weight; the other
            budget - recent are those of the largest weight, ties to the lowest
            position

    Kept rows move to the front in ascending order, their weights with them;
    freed places of `weights` become 0.  Returns (kept, new_lens): int32
    positions that stayed [num_seqs, num_kv_heads, budget] (-1 past the end) and
    int32 rows per sequence.  Pages past new_lens are free; sequences must not
    share pages.
    """
    d, bt = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    dev = k_cache.device
    cl = _t.as_i32(context_lens, dev).contiguous()
    budget, recent = int(budget), int(recent)
    assert cl.dim() == 1 and cl.shape[0] == bt.shape[0], "context_lens must be [num_seqs]"
    _t.require_cuda(weights)
    assert weights.dim() == 3 and weights.shape[:2] == (bt.shape[0], k_cache.shape[1]) \
        and weights.dtype == _torch.float32, "weights must be float32 [num_seqs, num_kv_heads, max_rows]"
    assert budget >= 1 and 0 <= recent <= budget, "budget must be >= 1 and recent in [0, budget]"
    kept = _torch.empty((bt.shape[0], k_cache.shape[1], budget), dtype=_torch.int32, device=dev)
    lens = _torch.empty((bt.shape[0],), dtype=_torch.int32, device=dev)
    _t.check(_t.lib().tak_kv8_evict(d, _t.ptr(cl), _t.ptr(weights), _t.strides(weights), weights.shape[2], budget,
                                    recent, _t.ptr(kept), _t.ptr(lens), _t.stream_of(k_cache)))
    return kept, lens
