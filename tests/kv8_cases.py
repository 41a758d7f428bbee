"""Seeded caches and tolerances shared by the 8-bit KV cache tests.

Tolerances, derived before the first run (u16 = 2^-8 for bf16, 2^-11 for fp16:
the unit roundoff of the output type, 2^-p for p bits of significand; e = 2^-24
that of fp32):

* rotary: one rounding of the result, plus products and cos / sin in fp32,
  at most 8 e of the pair's magnitude;
* codes, scales, kept rows, moved weights: equal;
* read-back: one rounding to the output type, one of the fp32 product;
* attention, with S the largest sum of |q k| / sqrt(D) over a row's keys and M
  the weighted sum of |v|: a score is off by at most ds = (D + 64) e S +
  16 e (|z| <= S), a weight by the factor exp(+-2 ds), so lse by ds + 8 e
  (1 + |lse|), and an output by u16 |o| + (2 ds + up) M, where up covers P held
  in 16 bits for the second product (2^-11), 2^-20 where it stays in fp32.
"""

import numpy as np
import torch

from oracle import kv8_oracle as K

E32 = 2.0 ** -24
ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E32}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def rng_of(*key):
    return np.random.default_rng(list(str(key).encode()))


def make(key, seqs, heads, block, group, dim, code, max_rows, spare=2, pool=None):
    """A cache full of rows N(0, size of the page and head), as an oracle Cache."""
    g = rng_of(key, seqs, heads, block, group, dim, code)
    width = -(-max_rows // block) if max_rows else 1
    nb = seqs * width + spare if pool is None else pool
    table = g.permutation(nb)[:seqs * width].reshape(seqs, width).astype(np.int32)
    codes, scales = [], []
    for _ in range(2):
        x = (g.standard_normal((nb, heads, block, dim)) * np.exp(g.standard_normal((nb, heads, 1, 1)))).astype(np.float32)
        y = x.reshape(nb, heads, block // group, group * dim)
        s = (np.abs(y).max(-1) * np.float32(1.0 / K.QMAX[code])).astype(np.float32)
        q = K.encode(y / s[..., None], code).reshape(x.shape).astype(np.float32)
        codes.append(q)
        scales.append(s)
    return K.Cache(code, codes, scales, table, group)


def to_device(c, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale, block_tables) on the device."""
    t = [torch.from_numpy(x).to(device).to(CODE[c.code]) for x in c.codes]
    s = [torch.from_numpy(x.copy()).to(device) for x in c.scales]
    return (*t, *s, torch.from_numpy(c.table).to(device))


def numbers(t):
    return t.float().cpu().numpy()


def same(c, dev):
    """The device's cache equals the oracle's, codes and scales (NaN scales too)."""
    for w in (0, 1):
        a, b = numbers(dev[w]), np.asarray(c.codes[w], np.float32)
        assert np.array_equal(a, b), f"plane {w}: {np.argwhere(a != b)[:4]} {a[a != b][:4]} {b[a != b][:4]}"
        assert np.array_equal(dev[2 + w].cpu().numpy(), c.scales[w], equal_nan=True)


def check_attention(got, want, dtype, dim, p16):
    out, lse, weights = got
    ref, rlse, rw, size, mass = want
    z = np.where(np.isfinite(rlse), np.abs(rlse), 0)
    ds = (dim + 64) * E32 * size + 16 * E32
    assert np.array_equal(np.isfinite(lse), np.isfinite(rlse))
    fin = np.isfinite(rlse)
    assert (np.abs(lse - rlse)[fin] <= (ds + 8 * E32 * (1 + z))[fin]).all(), np.abs(lse - rlse)[fin].max()
    tol = ULP[dtype] * np.abs(ref) + (2 * ds + p16)[..., None] * mass + 1e-30
    bad = np.abs(out - ref) > tol * 1.001 + (6e-8 if dtype == torch.float16 else 0)
    assert not bad.any(), (np.abs(out - ref)[bad].max(), np.argwhere(bad)[:4])
    if weights is not None:
        tol = (2 * ds.max() + 2.0 ** -20) * np.abs(rw) + 1e-12
        assert (np.abs(weights - rw) <= tol).all(), np.abs(weights - rw).max()
