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
_S3 = struct.Struct("=3q").pack
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
    """The C ABI's description of a cache (struct tak_kv8_cache, as bytes), the
    int32 block table that it points to, and (device index, num_kv_heads,
    head_dim, num_seqs)."""
    index = k_cache.get_device()
    assert index >= 0 and v_cache.get_device() == index and k_scale.get_device() == index \
        and v_scale.get_device() == index, "The cache's tensors must be on a CUDA device, all on the same"
    dtype = k_cache.dtype
    code = _CODES.get(dtype)
    assert code is not None, f"unsupported cache dtype {dtype}: expected int8 or float8_e4m3fn"
    shape = k_cache.shape
    assert len(shape) == 4 and v_cache.shape == shape and v_cache.dtype is dtype, \
        "k_cache and v_cache must be [num_blocks, num_kv_heads, block_size, head_dim] of one dtype"
    nb, hkv, rows, d = shape
    ss = k_scale.shape
    assert len(ss) == 3 and ss[0] == nb and ss[1] == hkv and v_scale.shape == ss, \
        "k_scale and v_scale must be [num_blocks, num_kv_heads, block_size / group]"
    assert k_scale.dtype is _torch.float32 and v_scale.dtype is _torch.float32, "scales must be float32"
    ng = ss[2]
    assert ng > 0 and rows % ng == 0, f"the number of scales ({ng}) must divide block_size ({rows})"
    bt = _t.i32_on(block_tables, index)
    assert bt.dim() == 2, "block_tables must be [num_seqs, max_blocks]"
    seqs, width = bt.shape
    return _PACK.pack(
        k_cache.data_ptr(), *k_cache.stride(), v_cache.data_ptr(), *v_cache.stride(),
        k_scale.data_ptr(), *k_scale.stride(), v_scale.data_ptr(), *v_scale.stride(),
        bt.data_ptr(), *bt.stride(), nb, hkv, rows, d, rows // ng, seqs, width, code), bt, (index, hkv, d, seqs)


def _lens(t, index, n, name):
    """A contiguous int32 [n] tensor on the device."""
    t = _t.i32_on(t, index)
    assert t.dim() == 1 and t.shape[0] == n, f"{name} must have {n} elements here"
    return t if t.is_contiguous() else t.contiguous()


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
    desc, _bt, (index, hkv, d, seqs) = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    shape = k.shape
    assert len(shape) == 3 and v.shape == shape and v.dtype is k.dtype, "K and V must have the same shape and dtype"
    assert k.get_device() == index and v.get_device() == index, "k / v must be on the cache's CUDA device"
    assert shape[1] == hkv and shape[2] == d, "k / v must be [total_tokens, num_kv_heads, head_dim] of the cache"
    start = _lens(start_lens, index, seqs, "start_lens")
    cu = None if cu_seqlens is None else _lens(cu_seqlens, index, seqs + 1, "cu_seqlens")
    assert cu is not None or shape[0] == seqs, "without cu_seqlens k / v hold one row per sequence"
    rc = _t.lib().tak_kv8_write(desc, k.data_ptr(), _S3(*k.stride()), v.data_ptr(), _S3(*v.stride()),
                                start.data_ptr(), None if cu is None else cu.data_ptr(), shape[0], _t.dtype_code(k),
                                _t.raw_stream(index))
    if rc:
        _t.check(rc)


def kv8_cache_read(k_cache, v_cache, k_scale, v_scale, block_tables, cu_seqlens, total_tokens, *,
                   start_lens=None, dtype=_torch.bfloat16):
    """Read rows back as fp16, bf16 or fp32: (k, v) [total_tokens,
    num_kv_heads, head_dim], rows cu_seqlens[s] and on holding positions
    start_lens[s] (None: 0) and on of sequence s.  Rows outside every sequence
    are zeros."""
    desc, _bt, (index, hkv, d, seqs) = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    cu = _lens(cu_seqlens, index, seqs + 1, "cu_seqlens")
    start = None if start_lens is None else _lens(start_lens, index, seqs, "start_lens")
    total = int(total_tokens)
    k = _torch.empty_strided((total, hkv, d), (hkv * d, d, 1), dtype=dtype, device=k_cache.device)
    v = _torch.empty_like(k)
    st = _S3(hkv * d, d, 1)
    rc = _t.lib().tak_kv8_read(desc, cu.data_ptr(), None if start is None else start.data_ptr(), total,
                               k.data_ptr(), st, v.data_ptr(), st, _t.dtype_code(k), _t.raw_stream(index))
    if rc:
        _t.check(rc)
    return k, v


def kv8_cache_evict(k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, weights, budget, recent):
    """Cut every sequence to at most `budget` rows per KV head, in place.

    Args:
        context_lens: [num_seqs] int32 rows that each sequence holds
        weights: [num_seqs, num_kv_heads, max_rows] float32 accumulated
            attention weights (paged_attention_kv8's `weights`); rows past
            max_rows weigh 0
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
    desc, _bt, (index, hkv, _d, seqs) = describe(k_cache, v_cache, k_scale, v_scale, block_tables)
    cl = _lens(context_lens, index, seqs, "context_lens")
    budget, recent = int(budget), int(recent)
    ws = weights.shape
    assert len(ws) == 3 and ws[0] == seqs and ws[1] == hkv and weights.dtype is _torch.float32, \
        "weights must be float32 [num_seqs, num_kv_heads, max_rows]"
    assert weights.get_device() == index, "weights must be on the cache's CUDA device"
    assert budget >= 1 and 0 <= recent <= budget, "budget must be >= 1 and recent in [0, budget]"
    kept = cl.new_empty((seqs, hkv, budget))
    lens = cl.new_empty((seqs,))
    rc = _t.lib().tak_kv8_evict(desc, cl.data_ptr(), weights.data_ptr(), _S3(*weights.stride()), ws[2], budget,
                                recent, kept.data_ptr(), lens.data_ptr(), _t.raw_stream(index))
    if rc:
        _t.check(rc)
    return kept, lens
