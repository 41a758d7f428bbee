"""Attention over the 8-bit cache where V's scales lie at the ends of their range (GPU).

Tolerances, derived before the first run (E32 = 2^-24).  Beside what
kv8_cases.py derives, a tensor-core weight is 2^(s + log2 vs + 13 - M): sums of
magnitudes up to 2 A each, A the largest |log2 vs| + 13 + |s| in base-2 units,
so four roundings put 8 A E32 on the exponent, and M + 10 + log2 l puts three
more, 6 A E32, on the log-sum-exp.  dv = 16 A E32 bounds both; outputs get 2 dv
of the row's mass.  2^-133 is a bf16 subnormal's spacing.
"""

import numpy as np
import pytest
import torch

import _tak_b200 as T
import kv8_cases as KC
from paged_attention_kv8 import paged_attention_kv8
from test_gpu_kv8 import dev32

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
LEAST = {"int8": 2.0 ** -100 / 127, "e4m3": 2.0 ** -100 / 448}  # the smallest scales that a write makes

SHAPES = [  # seqs, q heads, kv heads, dim, block, group, contexts, queries
    (2, 4, 1, 128, 32, 16, [300, 33], 1),
    (1, 8, 2, 64, 16, 16, [700], 1),
    (2, 16, 1, 128, 64, 32, [257, 16], 1),
    (1, 8, 1, 64, 16, 16, [500], 4),
    (1, 10, 2, 256, 32, 16, [200], 1),
    (1, 12, 1, 256, 32, 16, [200], 3),
    (64, 16, 8, 64, 16, 16, [200 - i for i in range(64)], 1),  # items of two chunks inside one CTA
    (64, 96, 8, 64, 16, 16, [200 - i for i in range(64)], 1),
]


def cache_of(key, i, code):
    """A cache without a code of 0, so that every column of a row has the mass of its heaviest keys."""
    seqs, _, hkv, dim, block, group, ctx, _ = SHAPES[i]
    c = KC.make((key, i), seqs, hkv, block, group, dim, code, max(ctx))
    for x in c.codes:
        x[x == 0] = 1
    return c


def check(c, i, path):
    seqs, H, hkv, dim, block, group, ctx, Lq = SHAPES[i]
    q = torch.randn(seqs, Lq, H, dim, generator=torch.Generator().manual_seed(i)).to(BF)
    d = KC.to_device(c)
    weights = torch.zeros(seqs, hkv, c.table.shape[1] * block, device=DEV)
    old = T.set_kernel_path(path)
    try:
        out, lse = paged_attention_kv8(q.to(DEV), *d, dev32(ctx), weights=weights, return_lse=True)
    finally:
        T.set_kernel_path(old)
    assert T.last_kernel() == ("kv8_attention_generic" if path else "kv8_attention_tc")
    ref, rlse, rw, size, mass = c.attend(q.double().numpy(), ctx)
    out, lse, got_w = KC.numbers(out).astype(np.float64), lse.cpu().double().numpy(), weights.cpu().double().numpy()
    ds = (dim + 64) * KC.E32 * size + 16 * KC.E32 + 16 * (135 + 1.5 * size) * KC.E32
    fin = np.isfinite(rlse)
    assert np.array_equal(np.isfinite(lse), fin)
    assert (np.abs(lse[fin] - rlse[fin]) <= (ds + 8 * KC.E32 * (1 + np.abs(np.where(fin, rlse, 0))))[fin]).all(), \
        np.abs(lse[fin] - rlse[fin]).max()
    tol = (2 * ds.max() + 2.0 ** -20) * np.abs(rw) + 1e-12
    assert (np.abs(got_w - rw) <= tol).all(), np.abs(got_w - rw).max()
    tol = KC.ULP[BF] * 1.001 * np.abs(ref) + (2 * ds + 2.0 ** -11)[..., None] * mass + 2.0 ** -133
    bad = ~(np.abs(out - ref) <= tol)
    assert not bad.any(), (bad.sum(), out[bad][:4], ref[bad][:4])


@pytest.mark.parametrize("path", [0, 1])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_smallest_v_scales(i, code, path):
    """Every V group at the smallest scales that a write makes."""
    c = cache_of("least", i, code)
    g = np.random.default_rng(i)
    c.scales[1][:] = (LEAST[code] * 2.0 ** g.uniform(0, 1.8, c.scales[1].shape)).astype(np.float32)
    check(c, i, path)


KINDS = {  # scales of V's groups; one in `every` is `odd`, the others `usual` (exponents of 2, or 0)
    "zeros beside large": (3, None, (36, 60)),
    "few zeros beside large": (7, None, (36, 60)),
    "small beside large": (2, (-100, -80), (40, 90)),
    "few large": (9, (60, 100), (-4, 4)),
    "all over": (2, (-108, 100), (-108, 100)),
    "all zero but few": (5, (-3, 90), None),
}


@pytest.mark.parametrize("path", [0, 1])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_v_scales_far_apart(i, kind, code, path):
    """Every key counts in the softmax whatever its group's V scale is beside
    the others'; scales of 0 among them."""
    c = cache_of(kind, i, code)
    every, odd, usual = KINDS[kind]
    g = np.random.default_rng(i)

    def draw(span):
        z = np.zeros(c.scales[1].shape)
        return z if span is None else 2.0 ** g.uniform(*span, z.shape)

    c.scales[1][:] = np.where(g.integers(0, every, c.scales[1].shape) == 0, draw(odd), draw(usual)).astype(np.float32)
    check(c, i, path)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_largest_values_on_cuda_cores(i, code):
    """Sums of values near fp32's largest stay finite before they are divided by the softmax's sum."""
    c = cache_of("most", i, code)
    top = 120 if code == "int8" else 118
    c.scales[1][:] = (2.0 ** np.random.default_rng(i).uniform(top - 14, top, c.scales[1].shape)).astype(np.float32)
    check(c, i, 1)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_largest_v_scales(i, code):
    """Values up to 2^127: the softmax's sum, in units of the largest value, is
    near fp32's smallest numbers."""
    c = cache_of("most", i, code)
    top = 120 if code == "int8" else 118
    c.scales[1][:] = (2.0 ** np.random.default_rng(i).uniform(top - 14, top, c.scales[1].shape)).astype(np.float32)
    check(c, i, 0)


def test_zero_v_scale_beside_a_large_one():
    """Two keys of equal scores, V of one zero and of the other large: half of the large one."""
    c = KC.make("half", 1, 1, 16, 16, 64, "int8", 32)
    c.codes[0][:] = 1
    c.scales[0][:] = 1
    c.scales[1][c.table[0, 0]] = 0
    c.scales[1][c.table[0, 1]] = 2.0 ** 40
    c.codes[1][c.table[0, 1]] = 100
    d = KC.to_device(c)
    q = torch.ones(1, 4, 64, dtype=BF, device=DEV)
    weights = torch.zeros(1, 1, 32, device=DEV)
    out = paged_attention_kv8(q, *d, dev32([32]), weights=weights)
    assert (out.float().cpu() / (50 * 2.0 ** 40) - 1).abs().max().item() < 2.0 ** -8
    assert (weights.cpu() * 8 - 1).abs().max().item() < 1e-5
