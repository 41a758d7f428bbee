"""Eviction from the 8-bit cache at the ends of its documented range (GPU)."""

import numpy as np
import pytest
import torch

import _tak_b200 as T
import kv8_cache as C8
import kv8_cases as KC
from test_gpu_kv8 import dev32

pytestmark = pytest.mark.gpu
DEV = "cuda"


def compare(c, ctx, w, budget, recent):
    """The device's eviction against the oracle's, all outputs equal."""
    d = KC.to_device(c)
    dw = torch.from_numpy(w.copy()).to(DEV)
    kept, lens = C8.kv8_cache_evict(*d, dev32(ctx), dw, budget, recent)
    rk, rl = c.evict(ctx, w, budget, recent)
    assert np.array_equal(lens.cpu().numpy(), rl) and np.array_equal(kept.cpu().numpy(), rk)
    assert np.array_equal(dw.cpu().numpy(), w, equal_nan=True)
    KC.same(c, d)


WIDE = [  # seqs, heads, block, group, dim, contexts, budget, recent
    (2, 2, 256, 256, 384, [700, 250], 300, 7),
    (1, 2, 256, 256, 512, [600], 257, 0),
    (2, 1, 256, 256, 640, [513, 700], 511, 100),
    (1, 1, 192, 192, 576, [500], 200, 5),
    (1, 2, 384, 192, 640, [700], 390, 390),
    (1, 1, 256, 256, 639, [600], 300, 10),   # no 16-byte pieces
    (1, 2, 256, 256, 384, [5000], 4500, 50),  # two windows for each CTA of a cluster
    (2, 40, 256, 256, 384, [600, 590], 520, 20),  # three windows for a CTA
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("i", range(len(WIDE)))
def test_evict_wide_groups(i, code):
    """Groups times head dims whose windows fill shared memory: both planes, weights and lengths agree."""
    seqs, heads, block, group, dim, ctx, budget, recent = WIDE[i]
    c = KC.make(("wide", i), seqs, heads, block, group, dim, code, max(ctx))
    w = (np.random.default_rng(i).random((seqs, heads, c.table.shape[1] * block)) ** 8).astype(np.float32)
    compare(c, ctx, w, budget, recent)


def test_refused_evictions_change_nothing():
    """Codes, scales, weights, kept and new_lens are as they were after each refusal."""
    c = KC.make("refuse", 2, 2, 512, 16, 64, "int8", 900)
    d = KC.to_device(c)
    w = torch.rand(2, 2, 1024, device=DEV)
    kept = torch.full((2, 2, 100), 7, dtype=torch.int32, device=DEV)
    lens = torch.full((2,), 7, dtype=torch.int32, device=DEV)
    ctx = dev32([900, 20])
    odd = torch.ones(*d[2].shape[:2], 1, device=DEV)  # one scale for 512 rows
    before = [t.clone() for t in (*d, w, kept, lens)]

    def call(cache, budget, recent):
        desc, _bt, _ = C8.describe(*cache)
        return T.lib().tak_kv8_evict(desc, ctx.data_ptr(), w.data_ptr(), T.strides(w), 1024, budget, recent,
                                     kept.data_ptr(), lens.data_ptr(), None)

    assert call((d[0], d[1], odd, odd, d[4]), 100, 10) == 1
    assert call(d, 0, 0) == 1 and call(d, 100, 101) == 1 and call(d, 1 << 31, 10) == 1
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (*d, w, kept, lens)))


NARROW = [  # rows, width of weights, budget, recent
    (700, 300, 200, 50), (700, 650, 200, 100), (700, 699, 300, 1), (700, 100, 400, 0), (700, 0, 300, 20),
    (700, 0, 300, 0), (700, 0, 300, 300), (700, 256, 700, 10), (700, 5, 699, 3), (30000, 9000, 12000, 100),
    (30000, 29999, 500, 0), (140001, 20000, 30000, 77), (200000, 150000, 1000, 10)]


@pytest.mark.parametrize("kind", ["spread", "ties", "negative", "nan"])
@pytest.mark.parametrize("i", range(len(NARROW)))
def test_evict_weights_narrower_than_the_context(i, kind):
    """Rows past `weights` count as weight 0: the newest stay, none is lost."""
    rows, width, budget, recent = NARROW[i]
    c = KC.make(("narrow", i), 2, 1, 64, 16, 16, "int8", rows)
    g = np.random.default_rng(i)
    w = (g.random((2, 1, width)) ** 8).astype(np.float32)
    if kind == "ties":
        w = np.round(w * 2).astype(np.float32)
        w[w == 0] = np.where(g.random((w == 0).sum()) < 0.5, 0.0, -0.0)
    if kind == "negative":  # rows without a weight rank above these
        w = -w - np.float32(1)
    if kind == "nan":
        w[g.random(w.shape) < 0.1] = np.nan
    compare(c, [rows, rows // 2], w, budget, recent)


def test_evict_budget_of_all_that_32_bits_hold():
    """No limit, written as the largest budget: every row stays, and kept is filled to its end."""
    c = KC.make("nolimit", 1, 1, 16, 16, 64, "int8", 50)
    d = KC.to_device(c)
    before = [t.clone() for t in d]
    w = torch.rand(1, 1, 64, device=DEV)
    budget = 2 ** 31 - 1
    kept, lens = C8.kv8_cache_evict(*d, dev32([50]), w, budget, 3)
    assert kept.shape == (1, 1, budget) and lens.tolist() == [50]
    assert kept[0, 0, :50].tolist() == list(range(50))
    for part in kept[0, 0, 50:].split(1 << 28):
        assert bool((part == -1).all())
    assert all(torch.equal(a, b) for a, b in zip(before, d))
