"""Rotary positions with several axes (time, height, width, ...) on B200.

An addition without a counterpart in suluner/triton-ascend-kernels: what a
model does to queries and keys before the attention modules of this folder.
"""

import ctypes

import _tak_b200 as _t


def rotary_nd(q, k, positions, inv_freq, sections, *, interleaved=False, inverse=False, out=None):
    """Turn the pairs of q's and k's heads by their tokens' positions.

    Args:
        q: [total_tokens, num_q_heads, head_dim]
        k: [total_tokens, num_kv_heads, head_dim], or None
        positions: [total_tokens, num_axes] integer positions ([total_tokens]
            for one axis)
        inv_freq: [rot_dim / 2] float32, radians per position of each pair
        sections: num_axes pair counts that add up to rot_dim / 2; pair i
            belongs to the axis in whose section it lies
        interleaved: pairs are (2i, 2i + 1) instead of (i, i + rot_dim / 2)
        inverse: turn the other way.  The rotation is orthogonal, so this is
            its gradient: grad_q, grad_k = rotary_nd(grad_out_q, grad_out_k,
            ..., inverse=True)
        out: (q_out, k_out) to write to; (q, k) turns them in place

    Returns ``(q_out, k_out)`` (k_out None without k).  Elements of a head past
    rot_dim are copied.
    """
    _t.require_cuda(q, k, positions, inv_freq)
    assert q.dim() == 3 and (k is None or k.dim() == 3), "q and k must be [total_tokens, num_heads, head_dim]"
    T, H, D = q.shape
    assert k is None or (k.shape[0] == T and k.shape[2] == D and k.dtype == q.dtype), \
        "k must have q's number of tokens, head_dim and dtype"
    pos = positions if positions.dim() == 2 else positions[:, None]
    sections = [int(x) for x in sections]
    assert pos.shape[0] == T and pos.shape[1] == len(sections), "positions must be [total_tokens, len(sections)]"
    assert inv_freq.dim() == 1 and inv_freq.dtype == _t.torch.float32 and inv_freq.shape[0] == sum(sections), \
        "inv_freq must be float32 with sum(sections) elements"
    assert 2 * sum(sections) <= D, f"rot_dim ({2 * sum(sections)}) exceeds head_dim ({D})"
    if pos.dtype != _t.torch.int32:
        pos = pos.to(_t.torch.int32)
    inv_freq = inv_freq.contiguous()
    qo, ko = out if out is not None else (q.new_empty(q.shape), None if k is None else k.new_empty(k.shape))
    for x, y in ((q, qo), (k, ko)):
        if x is not None:
            _t.require_cuda(y)
            assert y is not None and y.shape == x.shape and y.dtype == x.dtype, "out must match q and k"
    z = k is not None
    _t.check(_t.lib().tak_rotary_nd(
        _t.ptr(q), _t.strides(q), _t.ptr(k), _t.strides(k) if z else None, _t.ptr(pos), _t.strides(pos),
        _t.ptr(inv_freq), (ctypes.c_int32 * len(sections))(*sections), len(sections), _t.ptr(qo), _t.strides(qo),
        _t.ptr(ko) if z else None, _t.strides(ko) if z else None, T, H, k.shape[1] if z else 0, D,
        2 * sum(sections), int(bool(interleaved)), int(bool(inverse)), _t.dtype_code(q), _t.stream_of(q)))
    return qo, ko
