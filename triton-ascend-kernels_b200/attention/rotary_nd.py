"""Rotary positions with several axes (time, height, width, ...) on B200.

An addition without a counterpart in suluner/triton-ascend-kernels: what a
model does to queries and keys before the attention modules of this folder.
"""

import struct

import _tak_b200 as _t

_torch = _t.torch
_S2, _S3 = struct.Struct("=2q").pack, struct.Struct("=3q").pack
_SECTIONS = [struct.Struct(f"={n}i").pack for n in range(9)]


def rotary_nd(q, k, positions, inv_freq, sections, *, interleaved=False, inverse=False, out=None):
    """Turn the pairs of q's and k's heads by their tokens' positions.

    Args:
        q: [total_tokens, num_q_heads, head_dim]
        k: [total_tokens, num_kv_heads, head_dim], or None
        positions: [total_tokens, num_axes] integer positions ([total_tokens]
            for one axis)
        inv_freq: [rot_dim / 2] float32, radians per position of each pair
        sections: num_axes (at most 8) pair counts that add up to rot_dim / 2;
            pair i belongs to the axis in whose section it lies
        interleaved: pairs are (2i, 2i + 1) instead of (i, i + rot_dim / 2)
        inverse: turn the other way.  The rotation is orthogonal, so this is
            its gradient: grad_q, grad_k = rotary_nd(grad_out_q, grad_out_k,
            ..., inverse=True)
        out: (q_out, k_out) to write to; (q, k) turns them in place

    Returns ``(q_out, k_out)`` (k_out None without k).  Elements of a head past
    rot_dim are copied.
    """
    index = q.get_device()
    assert index >= 0 and positions.get_device() == index and inv_freq.get_device() == index, \
        "Tensors must be on a CUDA device, all on the same"
    shape = q.shape
    assert len(shape) == 3, "q must be [total_tokens, num_heads, head_dim]"
    T, H, D = shape
    dtype = q.dtype
    pos = positions if positions.dim() == 2 else positions[:, None]
    axes, pairs = len(sections), sum(sections)
    assert pos.shape == (T, axes), "positions must be [total_tokens, len(sections)]"
    assert inv_freq.dtype is _torch.float32 and inv_freq.shape == (pairs,), \
        "inv_freq must be float32 with sum(sections) elements"
    assert 2 * pairs <= D, f"rot_dim ({2 * pairs}) exceeds head_dim ({D})"
    if pos.dtype is not _torch.int32:
        assert not pos.is_floating_point() and not pos.is_complex(), \
            f"positions must be integers, not {pos.dtype} (fractions would be cut off)"
        pos = pos.to(_torch.int32)
    if not inv_freq.is_contiguous():
        inv_freq = inv_freq.contiguous()
    qo, ko = (_t.like(q), None) if out is None else out
    Hk, kp, ks, kop, kos = 0, None, None, None, None
    if k is not None:
        kshape = k.shape
        assert len(kshape) == 3 and kshape[0] == T and kshape[2] == D and k.dtype is dtype, \
            "k must have q's number of tokens, head_dim and dtype"
        assert k.get_device() == index, "k must be on q's device (CUDA)"
        Hk = kshape[1]
        if out is None:
            ko = _t.like(k)
        kp, ks, kop, kos = k.data_ptr(), _S3(*k.stride()), ko.data_ptr(), _S3(*ko.stride())
    if out is not None:
        for x, y in ((q, qo), (k, ko)):
            if x is not None:
                assert y is not None and y.get_device() == index and y.shape == x.shape and y.dtype is dtype, \
                    "out must match q and k"
    rc = _t.lib().tak_rotary_nd(
        q.data_ptr(), _S3(*q.stride()), kp, ks, pos.data_ptr(), _S2(*pos.stride()), inv_freq.data_ptr(),
        (_SECTIONS[axes] if axes < 9 else struct.Struct(f"={axes}i").pack)(*sections), axes, qo.data_ptr(),
        _S3(*qo.stride()), kop, kos, T, H, Hk, D, 2 * pairs, 1 if interleaved else 0, 1 if inverse else 0,
        _t.dtype_code(q), _t.raw_stream(index))
    if rc:
        _t.check(rc)
    return qo, ko
