"""CPU-side checks of the rotary positions and the 8-bit KV cache: the oracle
against other arithmetic, and the refusals that need no device."""

import ctypes

import numpy as np
import pytest
import torch

import _tak_b200 as T
import kv8_cache as C8
import kv8_cases as KC
from oracle import kv8_oracle as K
from paged_attention_kv8 import paged_attention_kv8
from rotary_nd import rotary_nd


def test_e4m3_rounding_matches_torch():
    x = torch.cat([torch.randn(20000) * 100, torch.randn(2000) * 1e-2, torch.arange(-448, 449) / 2,
                   torch.tensor([0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 448.0])]).clamp(-448, 448)
    assert np.array_equal(K.e4m3_round(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())


def test_oracle_rotary_is_a_rotation():
    g = np.random.default_rng(0)
    x, pos = g.standard_normal((5, 2, 16)), g.integers(0, 100, (5, 2))
    inv = (10.0 ** -np.arange(6)).astype(np.float32)
    for il in (False, True):
        y = K.rotary(x, pos, inv, [2, 4], il)
        assert np.allclose(np.linalg.norm(y, axis=-1), np.linalg.norm(x, axis=-1))
        assert np.allclose(K.rotary(y, pos, inv, [2, 4], il, inverse=True), x)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_oracle_write_then_attend(code):
    """A cache written in two calls holds its rows to half a step, and attention
    over it is the softmax over those rows."""
    c = KC.make("cpu", 1, 1, 16, 16, 32, code, 48)
    x = np.random.default_rng(1).standard_normal((40, 1, 32)).astype(np.float32)
    for lo, hi in ((0, 20), (20, 40)):
        for w in (0, 1):
            c.write(w, x[lo:hi], [lo], [0, hi - lo])
    got = c.values(0, 0, 0, 40)
    step = np.repeat([c.scales[0][c.table[0, i], 0, 0] for i in range(3)], 16)[:40, None]
    # a row may be rounded twice (half a step each) where its group grew; e4m3's step at the top is 32
    assert (np.abs(got - x[:, 0]) <= step * (1.01 if code == "int8" else 33)).all()
    q = np.random.default_rng(2).standard_normal((1, 1, 1, 32))
    out, lse, w, _, _ = c.attend(q, [40])
    z = got @ q[0, 0, 0] / np.sqrt(32)
    p = np.exp(z) / np.exp(z).sum()
    assert np.allclose(out[0, 0, 0], p @ c.values(1, 0, 0, 40)) and np.allclose(lse[0, 0, 0], np.log(np.exp(z).sum()))
    assert np.allclose(w[0, 0, :40], p) and w[0, 0, 40:].sum() == 0


def test_oracle_evict_keeps_the_largest():
    c = KC.make("cpu-ev", 1, 1, 8, 4, 16, "int8", 32)
    before = c.values(0, 0, 0, 30)
    w = np.zeros((1, 1, 32), np.float32)
    w[0, 0, [3, 9, 20]] = [1, 3, 2]
    kept, lens = c.evict([30], w, 5, 2)
    assert kept[0, 0].tolist() == [3, 9, 20, 28, 29] and lens.tolist() == [5]
    step = np.array([c.scales[0][c.table[0, 0], 0, i // 4] for i in range(5)])[:, None]
    assert (np.abs(c.values(0, 0, 0, 5) - before[kept[0, 0]]) <= 0.501 * step).all()
    assert w[0, 0, :5].tolist() == [1, 3, 2, 0, 0] and not w[0, 0, 5:].any()


def test_cpu_tensors_refused():
    k, v, ks, vs = C8.kv8_alloc(4, 2, 32, 64, group=16, device="cpu")
    assert k.shape == (4, 2, 32, 64) and ks.shape == (4, 2, 2) and k.dtype == torch.int8
    bt, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64)
    for call in (lambda: rotary_nd(q, q, n, torch.ones(32), [32]),
                 lambda: C8.kv8_cache_write(q[:, :2], q[:, :2], k, v, ks, vs, bt, n),
                 lambda: C8.kv8_cache_read(k, v, ks, vs, bt, torch.zeros(3, dtype=torch.int32), 0),
                 lambda: C8.kv8_cache_evict(k, v, ks, vs, bt, n, torch.zeros(2, 2, 64), 8, 2),
                 lambda: paged_attention_kv8(q, k, v, ks, vs, bt, n)):
        with pytest.raises(AssertionError, match="CUDA"):
            call()
    with pytest.raises(AssertionError, match="dtype"):
        C8.kv8_alloc(4, 2, 32, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(AssertionError, match="group"):
        C8.kv8_alloc(4, 2, 32, 64, group=24, device="cpu")


def _cache(**over):
    d = dict(nb=4, hkv=2, block=16, dim=64, group=16, seqs=2, width=2, code=0)
    d.update(over)
    p = 4096  # never dereferenced: every call below is refused on the host
    return C8._PACK.pack(p, 1, 1, 1, 1, p, 1, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 1, p, 1, 1, d["nb"], d["hkv"], d["block"],
                         d["dim"], d["group"], d["seqs"], d["width"], d["code"])


def test_c_entry_points_refuse():
    import os
    if not os.path.exists(T.LIB_PATH):
        pytest.skip("libtak_b200.so not built")
    L = T.lib()
    assert C8._PACK.size == 8 * (5 + 5 + 4 + 4 + 3 + 8)
    st = (ctypes.c_int64 * 4)(1, 1, 1, 1)
    p = ctypes.c_void_p(4096)

    def attend(c, H=4, Lq=1, dtype=1, cap=0.0, q=p, width=0):
        return L.tak_kv8_attention(c, q, st, p, p, st, None, None, None, width, H, Lq, 1.0, cap, dtype, None, 0, None)

    def refused(rc, word):
        assert rc == 1, rc
        assert word in T.lib().tak_last_error().decode(), T.lib().tak_last_error().decode()

    for over, word in ((dict(code=2), "code type"), (dict(hkv=0), "num_kv_heads"), (dict(dim=641), "head_dim"),
                       (dict(block=0), "block_size"), (dict(group=0), "group"), (dict(group=24), "group"),
                       (dict(block=512, group=512), "group"), (dict(seqs=-1), "num_seqs"), (dict(nb=-1), "num_blocks"),
                       (dict(width=1 << 28), "max_blocks")):
        refused(attend(_cache(**over)), word)
        refused(L.tak_kv8_write(_cache(**over), p, st, p, st, p, None, 2, 1, None), word)
        refused(L.tak_kv8_read(_cache(**over), p, None, 2, p, st, p, st, 1, None), word)
        refused(L.tak_kv8_evict(_cache(**over), p, p, st, 32, 4, 2, p, p, None), word)
        assert L.tak_kv8_attention_workspace_size(_cache(**over), 4, 1, 0, 1) == -1
    refused(attend(None), "null cache")
    refused(attend(_cache(), H=3), "num_q_heads")
    refused(attend(_cache(), dtype=3), "dtype")
    refused(attend(_cache(), cap=-1.0), "softcap")
    refused(attend(_cache(), cap=float("nan")), "softcap")
    refused(attend(_cache(), q=None), "null")
    refused(attend(_cache(), width=-1), "weights_width")
    refused(L.tak_kv8_write(_cache(), p, st, p, st, p, None, 3, 1, None), "one row per sequence")
    refused(L.tak_kv8_write(_cache(), None, st, p, st, p, None, 2, 1, None), "null")
    refused(L.tak_kv8_read(_cache(seqs=0), p, None, 2, p, st, p, st, 1, None), "no sequence")
    refused(L.tak_kv8_evict(_cache(), p, p, st, 32, 0, 0, p, p, None), "budget")
    refused(L.tak_kv8_evict(_cache(), p, p, st, 32, 4, 5, p, p, None), "recent")
    sec = (ctypes.c_int32 * 2)(16, 16)

    def rotary(sections=sec, axes=2, T_=3, D=64, rot=64, dtype=1, q=p):
        return L.tak_rotary_nd(q, st, None, None, p, st, p, sections, axes, p, st, None, None, T_, 4, 0, D, rot, 0, 0,
                               dtype, None)

    refused(rotary(rot=62), "sections")
    refused(rotary(rot=63), "rot_dim")
    refused(rotary(D=32), "rot_dim")
    refused(rotary(axes=9), "axes")
    refused(rotary(dtype=7), "dtype")
    refused(rotary(q=None), "null q")
    refused(rotary(T_=-1), "total_tokens")
    refused(rotary((ctypes.c_int32 * 2)(-1, 33)), "negative")


def test_another_current_device_is_refused(monkeypatch):
    monkeypatch.setattr(T, "_current_device", lambda: 1)
    monkeypatch.setattr(T, "_raw_stream", lambda index: 40 + index)
    assert T.raw_stream(1) == 41
    with pytest.raises(AssertionError, match="current device"):
        T.raw_stream(0)
