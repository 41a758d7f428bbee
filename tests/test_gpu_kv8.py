"""Rotary positions and the 8-bit KV cache against 64-bit restatements (GPU)."""

import numpy as np
import pytest
import torch

import _tak_b200 as T
import kv8_cache as C8
import kv8_cases as KC
from oracle import kv8_oracle as K
from paged_attention_kv8 import paged_attention_kv8
from rotary_nd import rotary_nd

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def dev32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- rotary
def rot_inputs(seed, tokens, heads, kv_heads, dim, rot, axes, dtype, high=131072):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(tokens, heads, dim, generator=g).to(dtype)
    k = torch.randn(tokens, kv_heads, dim, generator=g).to(dtype)
    pos = torch.randint(0, high, (tokens, axes), generator=g, dtype=torch.int32)
    half = rot // 2
    sec = [half // axes] * axes
    sec[-1] += half - sum(sec)
    inv = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()
    return q, k, pos, inv, sec


def check_rot(y, x, pos, inv, sec, il, inverse):
    x64 = x.double().numpy()
    ref = K.rotary(x64, pos.numpy(), inv.numpy(), sec, il, inverse)
    # a pair's magnitude is kept by the rotation
    rot = 2 * sum(sec)
    i = np.arange(rot // 2)
    p, q = (2 * i, 2 * i + 1) if il else (i, i + rot // 2)
    size = np.zeros_like(ref)
    size[..., p] = size[..., q] = np.hypot(ref[..., p], ref[..., q])
    tol = KC.ULP[x.dtype] * 1.001 * np.abs(ref) + 8 * KC.E32 * size + (3.1e-8 if x.dtype == HF else 0)
    err = np.abs(y.double().cpu().numpy() - ref)
    assert (err <= tol).all(), (err.max(), np.argwhere(err > tol)[:3])
    assert np.array_equal(y.float().cpu().numpy()[..., rot:], x.float().numpy()[..., rot:])


@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,axes", [
    (1, 1, 1, 2, 2, 1), (1, 32, 8, 128, 128, 3), (67, 5, 1, 80, 64, 2), (33, 4, 4, 72, 72, 3), (130, 16, 2, 256, 96, 2),
    (9, 3, 1, 65, 30, 4), (64, 8, 8, 128, 0, 1), (257, 2, 2, 64, 64, 1)])
def test_rotary(dtype, il, tokens, heads, kv, dim, rot, axes):
    q, k, pos, inv, sec = rot_inputs(tokens + dim, tokens, heads, kv, dim, rot, axes, dtype)
    for inverse in (False, True):
        qo, ko = rotary_nd(q.to(DEV), k.to(DEV), pos.to(DEV), inv.to(DEV), sec, interleaved=il, inverse=inverse)
        check_rot(qo, q, pos, inv, sec, il, inverse)
        check_rot(ko, k, pos, inv, sec, il, inverse)


@pytest.mark.parametrize("il", [False, True])
def test_rotary_views_in_place_and_without_k(il):
    """q and k as slices of one projection's output, written in place; the
    elements between them stay; positions transposed; q alone."""
    q, k, pos, inv, sec = rot_inputs(5, 37, 6, 2, 64, 48, 3, BF)
    big = torch.randn(37, 12, 64).to(BF)
    big[:, :6], big[:, 7:9] = q, k
    keep = big.clone()
    b = big.to(DEV)
    qv, kv = b[:, :6], b[:, 7:9]
    rotary_nd(qv, kv, pos.t().contiguous().to(DEV).t(), inv.to(DEV), sec, interleaved=il, out=(qv, kv))
    check_rot(b[:, :6], q, pos, inv, sec, il, False)
    check_rot(b[:, 7:9], k, pos, inv, sec, il, False)
    assert torch.equal(b.cpu()[:, 6], keep[:, 6]) and torch.equal(b.cpu()[:, 9:], keep[:, 9:])
    qo, none = rotary_nd(q.to(DEV), None, pos.to(DEV), inv.to(DEV), sec, interleaved=il)
    assert none is None
    check_rot(qo, q, pos, inv, sec, il, False)
    # a transposed head axis: no element stride of 1
    qt = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    qo, _ = rotary_nd(qt, None, pos.to(DEV), inv.to(DEV), sec, interleaved=il)
    check_rot(qo, q, pos, inv, sec, il, False)
    # storage that starts off a 16-byte boundary
    qm = torch.empty(q.numel() + 1, dtype=BF, device=DEV)[1:].view(q.shape)
    qm.copy_(q)
    qo, _ = rotary_nd(qm, None, pos.to(DEV), inv.to(DEV), sec, interleaved=il)
    check_rot(qo, q, pos, inv, sec, il, False)


def test_rotary_one_axis_negative_positions_and_empty():
    q, k, pos, inv, sec = rot_inputs(6, 20, 2, 1, 64, 64, 1, FF)
    pos = -pos
    qo, _ = rotary_nd(q.to(DEV), k.to(DEV), pos[:, 0].to(DEV), inv.to(DEV), sec)
    check_rot(qo, q, pos, inv, sec, False, False)
    qo, ko = rotary_nd(q[:0].to(DEV), k[:0].to(DEV), pos[:0].to(DEV), inv.to(DEV), sec)
    assert qo.shape == (0, 2, 64) and ko.shape == (0, 1, 64)


@pytest.mark.parametrize("il", [False, True])
def test_rotary_inverse_is_the_gradient(il):
    """d/dx of sum(c * rotary(x)) is rotary_inverse(c): against central
    differences of the forward call in fp32, exact up to rounding as it is linear."""
    q, _, pos, inv, sec = rot_inputs(7, 5, 2, 1, 16, 12, 2, FF, high=50)
    c = torch.randn(5, 2, 16, generator=torch.Generator().manual_seed(1))
    grad, _ = rotary_nd(c.to(DEV), None, pos.to(DEV), inv.to(DEV), sec, interleaved=il, inverse=True)
    h, num = 0.5, torch.zeros_like(q)
    for d in range(16):
        e = torch.zeros_like(q)
        e[..., d] = h
        f = [rotary_nd((q + s * e).to(DEV), None, pos.to(DEV), inv.to(DEV), sec, interleaved=il)[0].cpu().double()
             for s in (1, -1)]
        num[..., d] = ((f[0] - f[1]) / (2 * h) * c.double()).sum(-1).float()
    # 16 products of rounded outputs, magnitudes below 8
    assert (grad.cpu() - num).abs().max().item() <= 16 * 2 * 8 * 8 * KC.E32


# ---------------------------------------------------------------- write and read
WRITE = [  # seqs, heads, block, group, dim, starts, counts
    (1, 1, 16, 16, 128, [0], [1]),
    (3, 2, 32, 16, 64, [0, 15, 16], [1, 1, 1]),
    (4, 2, 64, 32, 128, [0, 31, 33, 7], [70, 1, 64, 0]),
    (2, 3, 16, 4, 40, [3, 0], [21, 2]),
    (2, 1, 24, 12, 33, [5, 11], [30, 13]),
    (2, 2, 128, 128, 128, [100, 0], [60, 129]),
    (3, 1, 128, 64, 256, [0, 63, 64], [200, 1, 3]),
    (1, 1, 256, 256, 64, [17], [300]),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("i", range(len(WRITE)))
def test_write_and_read(i, dtype, code):
    seqs, heads, block, group, dim, starts, counts = WRITE[i]
    c = KC.make(("write", i), seqs, heads, block, group, dim, code, max(a + b for a, b in zip(starts, counts)))
    d = KC.to_device(c)
    cu = np.concatenate([[0], np.cumsum(counts)])
    g = torch.Generator().manual_seed(i)
    k, v = (torch.randn(cu[-1], heads, dim, generator=g).mul(m).to(dtype) for m in (1.0, 5.0))
    C8.kv8_cache_write(k.to(DEV), v.to(DEV), *d, dev32(starts), dev32(cu))
    for w, x in enumerate((k, v)):
        c.write(w, x.float().numpy(), starts, cu)
    KC.same(c, d)
    # written rows are within half a step of their inputs (int8)
    lens = [a + b for a, b in zip(starts, counts)]
    cr = np.concatenate([[0], np.cumsum(lens)])
    for dt in (BF, HF, FF):
        rk, rv = C8.kv8_cache_read(*d, dev32(cr), int(cr[-1]) + 2, dtype=dt)
        assert rk.dtype == dt and not rk[cr[-1]:].float().any() and not rv[cr[-1]:].float().any()
        for w, y in enumerate((rk, rv)):
            for s in range(seqs):
                for h in range(heads):
                    ref = c.values(w, s, h, lens[s])
                    err = np.abs(KC.numbers(y)[cr[s]:cr[s + 1], h] - ref)
                    assert (err <= (KC.ULP[dt] + KC.E32) * 1.001 * np.abs(ref) + 3e-8).all()
    if code == "int8":
        for s in range(seqs):
            for h in range(heads):
                got = c.values(0, s, h, lens[s])[starts[s]:]
                x = k[cu[s]:cu[s + 1], h].float().numpy()
                # the row's own group may later have grown no further, so half of its final step bounds it
                if counts[s]:
                    steps = np.array([c.scales[0][a[0], h, a[1] // group] for a in
                                      (c.at(s, r) for r in range(starts[s], lens[s]))])
                    assert (np.abs(got - x) <= 0.5 * steps[:, None] * (1 + 2e-5)).all()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_token_by_token(code):
    """Decode steps with one row per sequence, growing magnitudes: the open
    group is requantised at nearly every step."""
    c = KC.make("append", 3, 2, 32, 16, 64, code, 80)
    d = KC.to_device(c)
    starts = np.array([0, 13, 31], np.int32)
    g = torch.Generator().manual_seed(3)
    for step in range(36):
        k, v = (torch.randn(3, 2, 64, generator=g).mul(1.2 ** step).to(BF) for _ in range(2))
        C8.kv8_cache_write(k.to(DEV), v.to(DEV), *d, dev32(starts + step))
        for w, x in enumerate((k, v)):
            c.write(w, x.float().numpy(), (starts + step).tolist(), [0, 1, 2, 3])
    KC.same(c, d)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_zeros_tiny_inf_nan(code):
    """All-zero and tiny groups are zeros with scale 0; an infinity or a NaN
    makes its group's scale NaN, and a NaN scale stays."""
    c = KC.make("odd", 1, 1, 16, 16, 64, code, 96)
    d = KC.to_device(c)
    x = torch.randn(80, 1, 64, generator=torch.Generator().manual_seed(1))
    x[0:16] = 0
    x[16:32] *= 1e-33
    x[40, 0, 7] = float("inf")
    x[50, 0, 3] = float("nan")
    x[64:] *= 1e30
    for lo, hi in ((0, 45), (45, 80)):
        C8.kv8_cache_write(x[lo:hi].to(DEV), x[lo:hi].to(DEV), *d, dev32([lo]), dev32([0, hi - lo]))
        for w in (0, 1):
            c.write(w, x[lo:hi].numpy(), [lo], [0, hi - lo])
    KC.same(c, d)
    s = d[2].cpu().numpy()[c.table[0], 0, 0]
    assert s[0] == 0 and s[1] == 0 and np.isnan(s[2]) and np.isnan(s[3]) and np.isfinite(s[4])


def test_write_read_bad_pages_and_views():
    """Rows past the table or on pages outside the pool are dropped and read as
    zeros; caches, scales, inputs and tables may be strided views."""
    c = KC.make("views", 2, 2, 16, 16, 64, "int8", 64)
    pool = [torch.zeros(c.nb + 4, 3, 16, 64, dtype=torch.int8, device=DEV) for _ in range(2)]
    sc = [torch.zeros(c.nb + 4, 3, 1, device=DEV) for _ in range(2)]
    for w in range(2):
        pool[w][2:-2, :2] = torch.from_numpy(c.codes[w]).to(DEV).to(torch.int8)
        sc[w][2:-2, :2] = torch.from_numpy(c.scales[w]).to(DEV)
    before = [x.clone() for x in pool + sc]
    bad = c.table.copy()
    bad[0, 1], bad[1, 2] = c.nb, -1
    c.table = bad
    wide = torch.zeros(2, 6, dtype=torch.int32, device=DEV)
    wide[:, :4] = torch.from_numpy(bad).to(DEV)
    d = (pool[0][2:-2, :2], pool[1][2:-2, :2], sc[0][2:-2, :2], sc[1][2:-2, :2], wide[:, :4])
    x = torch.randn(2, 140, 64, generator=torch.Generator().manual_seed(2)).to(BF)
    kv = x.to(DEV).transpose(0, 1)  # [140, 2, 64], head axis outermost in memory
    C8.kv8_cache_write(kv, kv, *d, dev32([0, 3]), dev32([0, 70, 140]))
    for w in range(2):
        c.write(w, x.float().numpy().transpose(1, 0, 2), [0, 3], [0, 70, 140])
    KC.same(c, d)
    for t, b in zip(pool + sc, before):  # nothing outside the view moved
        assert torch.equal(t[:2], b[:2]) and torch.equal(t[-2:], b[-2:]) and torch.equal(t[:, 2], b[:, 2])
    rk, _ = C8.kv8_cache_read(*d, dev32([0, 70, 140]), 140, dtype=FF, start_lens=dev32([0, 3]))
    for s in range(2):
        for h in range(2):
            ref = c.values(0, s, h, 73)[3 * s:][:70]
            assert np.array_equal(rk[70 * s:70 * s + 70, h].cpu().numpy(), ref.astype(np.float32))


# ---------------------------------------------------------------- attention
ATT = [  # seqs, q heads, kv heads, dim, block, group, contexts, queries
    (1, 4, 1, 128, 16, 16, [1], 1),
    (2, 32, 8, 128, 16, 16, [17, 300], 1),
    (5, 8, 2, 64, 32, 16, [0, 1, 31, 64, 257], 1),
    (3, 16, 1, 128, 64, 64, [63, 65, 700], 1),
    (2, 40, 2, 128, 128, 32, [129, 511], 1),
    (2, 4, 2, 256, 32, 32, [33, 200], 1),
    (2, 6, 3, 96, 48, 48, [100, 47], 1),
    (3, 8, 2, 128, 16, 16, [2, 4, 90], 4),
    (2, 64, 2, 128, 64, 16, [129, 70], 3),
    (2, 5, 5, 40, 8, 4, [9, 30], 2),
    (2, 16, 2, 64, 128, 128, [128, 1000], 9),
    (1, 2, 1, 80, 16, 16, [333], 1),
    (2, 8, 8, 256, 64, 16, [260, 64], 5),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("i", range(len(ATT)))
@pytest.mark.parametrize("path", [0, 1])
def test_attention(i, dtype, code, path):
    seqs, H, hkv, dim, block, group, ctx, Lq = ATT[i]
    c = KC.make(("att", i), seqs, hkv, block, group, dim, code, max(ctx))
    d = KC.to_device(c)
    g = torch.Generator().manual_seed(i)
    q = torch.randn(seqs, Lq, H, dim, generator=g).to(dtype)
    cap = 0.0 if i % 2 else 20.0
    width = c.table.shape[1] * block if i % 3 else max(max(ctx) - 5, 1)
    weights = torch.rand(seqs, hkv, width, generator=g).to(DEV)
    start = weights.cpu().double().numpy()
    qd = (q if Lq > 1 else q[:, 0]).to(DEV)
    old = T.set_kernel_path(path)
    try:
        out, lse = paged_attention_kv8(qd, *d, dev32(ctx), softcap=cap, weights=weights, return_lse=True)
        plain = paged_attention_kv8(qd, *d, dev32(ctx), softcap=cap)
    finally:
        T.set_kernel_path(old)
    assert out.shape == qd.shape and lse.shape == qd.shape[:-1]
    assert torch.equal(out, plain)  # the weights change nothing else
    want = c.attend(q.double().numpy(), ctx, cap, width)
    shape = (seqs, Lq, H)
    p16 = 2.0 ** -11 if T.last_kernel() != "kv8_attention_generic" else 2.0 ** -20
    got_w = weights.cpu().double().numpy() - start
    KC.check_attention((KC.numbers(out).reshape(*shape, dim).astype(np.float64),
                        lse.cpu().double().numpy().reshape(shape), None), want, dtype, dim, p16)
    ds = (dim + 64) * KC.E32 * want[3].max() + 16 * KC.E32
    assert (np.abs(got_w - want[2]) <= (2 * ds + 2.0 ** -20) * want[2] + 2.0 ** -22 * (start + want[2])).all()
    assert T.read_device_error() == 0


@pytest.mark.parametrize("path", [0, 1])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_stale_rows_bad_pages_and_views(code, path):
    """Codes and scales after a sequence's end are never used, NaN among them;
    pages outside the pool count as zero rows; q, out and cache strides."""
    c = KC.make("stale", 3, 2, 32, 16, 128, code, 200)
    ctx = [40, 200, 7]
    tab = c.table.copy()
    tab[1, 2], tab[1, 4] = -1, c.nb + 3
    c.table = tab
    want_cache = KC.to_device(c)
    for s, n in enumerate(ctx):  # poison what lies past the end
        for r in range(n, c.table.shape[1] * 32):
            a = c.at(s, r)
            if a:
                for w in range(2):
                    t = want_cache[w]
                    t.view(torch.int8)[a[0], :, a[1]] = 0x7f if code == "e4m3" else -127
                    if a[1] % 16 == 0:
                        want_cache[2 + w][a[0], :, a[1] // 16] = float("nan")
    q = torch.randn(3, 4, 1, 128, generator=torch.Generator().manual_seed(4)).to(BF)
    big = torch.zeros(3, 9, 128, dtype=BF, device=DEV)
    big[:, 3:7] = q[:, :, 0].to(DEV)
    old = T.set_kernel_path(path)
    try:
        out, lse = paged_attention_kv8(big[:, 3:7], *want_cache, dev32(ctx), return_lse=True)
    finally:
        T.set_kernel_path(old)
    want = c.attend(q[:, :, 0].double().numpy()[:, None], ctx)
    KC.check_attention((KC.numbers(out)[:, None].astype(np.float64), lse.cpu().double().numpy()[:, None], None), want,
                       BF, 128, 2.0 ** -11)


@pytest.mark.parametrize("path", [0, 1])
def test_attention_extreme_scales_and_queries(path):
    """V scales many orders apart (a large V under a vanishing weight must not
    drown a small V under a large one), scales of 0, and large and tiny queries."""
    c = KC.make("scales", 1, 1, 64, 16, 64, "int8", 128)
    g = np.random.default_rng(5)
    c.scales[1][:] = 10.0 ** g.uniform(-12, 3, c.scales[1].shape).astype(np.float32)
    c.scales[1][c.table[0, 0], 0, 1] = 0
    c.scales[0][c.table[0, 1], 0, 2] = 0
    q = torch.randn(1, 1, 4, 64, generator=torch.Generator().manual_seed(4)) * torch.tensor([1e-6, 1.0, 30.0, 3e3])[:, None]
    d = KC.to_device(c)
    old = T.set_kernel_path(path)
    try:
        for dtype in (BF, FF):
            qd = q.to(dtype)
            out, lse = paged_attention_kv8(qd.to(DEV), *d, dev32([128]), return_lse=True)
            want = c.attend(qd.double().numpy(), [128])
            KC.check_attention((KC.numbers(out).astype(np.float64), lse.cpu().double().numpy(), None), want, dtype, 64,
                               2.0 ** -11)
    finally:
        T.set_kernel_path(old)


@pytest.mark.parametrize("path", [0, 1])
def test_attention_nan_and_inf_reach_only_their_rows(path):
    c = KC.make("nan", 2, 2, 32, 32, 128, "int8", 64)
    c.scales[0][c.table[0, 1], 1, 0] = np.nan
    d = KC.to_device(c)
    q = torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(4)).to(BF)
    q[1, 0, 5] = float("nan")
    old = T.set_kernel_path(path)
    try:
        out = paged_attention_kv8(q.to(DEV), *d, dev32([60, 33])).float().cpu()
    finally:
        T.set_kernel_path(old)
    bad = torch.isnan(out).all(-1)
    assert bad.tolist() == [[False, False, True, True], [True, False, False, False]]
    assert torch.isfinite(out[~bad]).all()


def test_attention_on_another_stream_and_twice():
    c = KC.make("stream", 4, 2, 64, 16, 128, "int8", 900)
    d = KC.to_device(c)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(9)).to(BF).to(DEV)
    ctx = dev32([900, 1, 450, 899])
    a = paged_attention_kv8(q, *d, ctx)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        b = paged_attention_kv8(q, *d, ctx)
    st.synchronize()
    assert torch.equal(a, b)  # the same bits again: nothing depends on an order of arrival
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        paged_attention_kv8(q, *d, ctx)
    st.synchronize()
    with torch.cuda.graph(g, stream=st):
        e = paged_attention_kv8(q, *d, ctx)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, e)


# ---------------------------------------------------------------- eviction
EV = [  # seqs, heads, block, group, dim, contexts, budget, recent
    (1, 1, 16, 16, 64, [40], 17, 5),
    (3, 2, 32, 16, 128, [0, 20, 200], 20, 0),
    (2, 2, 64, 64, 128, [300, 65], 64, 64),
    (2, 1, 8, 4, 33, [50, 9], 1, 1),
    (2, 2, 128, 32, 64, [3000, 2500], 1037, 100),
    (1, 2, 256, 256, 64, [700], 300, 7),
    (2, 1, 16, 16, 256, [128, 600], 128, 16),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("i", range(len(EV)))
def test_evict(i, kind, code):
    seqs, heads, block, group, dim, ctx, budget, recent = EV[i]
    c = KC.make(("evict", i), seqs, heads, block, group, dim, code, max(ctx))
    d = KC.to_device(c)
    g = np.random.default_rng(i)
    width = c.table.shape[1] * block
    w = g.random((seqs, heads, width)).astype(np.float32) ** 8
    if kind == "ties":
        w = np.round(w * 3).astype(np.float32)
        w[w == 0] = np.where(g.random((w == 0).sum()) < 0.5, 0.0, -0.0)
    if kind == "odd":
        w *= np.where(g.random(w.shape) < 0.5, -1, 1).astype(np.float32)
        w[g.random(w.shape) < 0.05] = np.nan
        w[g.random(w.shape) < 0.05] = np.inf
        w[g.random(w.shape) < 0.05] = -np.inf
    dw = torch.from_numpy(w.copy()).to(DEV)
    kept, lens = C8.kv8_cache_evict(*d, dev32(ctx), dw, budget, recent)
    rk, rl = c.evict(ctx, w, budget, recent)
    assert np.array_equal(lens.cpu().numpy(), rl)
    assert np.array_equal(kept.cpu().numpy(), rk)
    assert np.array_equal(dw.cpu().numpy(), w, equal_nan=True)
    KC.same(c, d)


def test_evict_views_and_bad_pages():
    c = KC.make("evv", 2, 2, 16, 16, 64, "e4m3", 160)
    c.table[0, 3], c.table[1, 1] = -5, c.nb
    d = KC.to_device(c)
    w = np.random.default_rng(0).random((2, 2, 320)).astype(np.float32)
    dw = torch.from_numpy(w.copy()).to(DEV)
    kept, lens = C8.kv8_cache_evict(*d, dev32([150, 400]), dw[:, :, ::2], 70, 10)  # 400 rows asked of a table for 160
    v = w[:, :, ::2].copy()
    rk, rl = c.evict([150, 400], v, 70, 10)
    assert np.array_equal(kept.cpu().numpy(), rk) and lens.tolist() == [70, 70]
    w[:, :, ::2] = v
    assert np.array_equal(dw.cpu().numpy(), w)
    KC.same(c, d)


# ---------------------------------------------------------------- refusals
def test_refusals():
    c = KC.make("ref", 2, 2, 16, 16, 64, "int8", 32)
    k, v, ks, vs, bt = KC.to_device(c)
    q = torch.zeros(2, 4, 64, dtype=BF, device=DEV)
    ctx = dev32([3, 4])
    A = AssertionError
    for bad in (lambda: paged_attention_kv8(q.cpu(), k, v, ks, vs, bt, ctx),
                lambda: paged_attention_kv8(q[:, :3], k, v, ks, vs, bt, ctx),
                lambda: paged_attention_kv8(q[..., :32], k, v, ks, vs, bt, ctx),
                lambda: paged_attention_kv8(q, k, v[:, :1], ks, vs, bt, ctx),
                lambda: paged_attention_kv8(q, k, v, ks.double(), vs, bt, ctx),
                lambda: paged_attention_kv8(q, k.to(torch.int16), v.to(torch.int16), ks, vs, bt, ctx),
                lambda: paged_attention_kv8(q, k, v, ks, vs, bt[:1], ctx),
                lambda: paged_attention_kv8(q, k, v, ks, vs, bt, ctx[:1]),
                lambda: paged_attention_kv8(q, k, v, ks, vs, bt, ctx, softcap=-1.0),
                lambda: paged_attention_kv8(q, k, v, ks, vs, bt, ctx, weights=torch.zeros(2, 2, 8, device=DEV).half()),
                lambda: C8.kv8_cache_write(q[:, :2], q[:, :2], k, v, ks, vs, bt, ctx[:1]),
                lambda: C8.kv8_cache_write(q, q, k, v, ks, vs, bt, ctx),
                lambda: C8.kv8_cache_write(q[:1, :2], q[:1, :2], k, v, ks, vs, bt, ctx),
                lambda: C8.kv8_cache_read(k, v, ks, vs, bt, dev32([0, 3]), 3),
                lambda: C8.kv8_cache_evict(k, v, ks, vs, bt, ctx, torch.zeros(2, 2, 8, device=DEV), 4, 5),
                lambda: C8.kv8_cache_evict(k, v, ks, vs, bt, ctx, torch.zeros(2, 2, 8, device=DEV), 0, 0),
                lambda: rotary_nd(q, None, ctx, torch.ones(32, device=DEV), [16, 16]),
                lambda: rotary_nd(q, None, ctx, torch.ones(33, device=DEV), [33]),
                lambda: rotary_nd(q, q[:1], ctx, torch.ones(32, device=DEV), [32])):
        with pytest.raises(A):
            bad()
    with pytest.raises(TypeError):
        paged_attention_kv8(q.double(), k, v, ks, vs, bt, ctx)
    with pytest.raises(RuntimeError, match="1 to 8 axes"):
        rotary_nd(q, None, ctx[:, None].expand(2, 9), torch.ones(9, device=DEV), [1] * 9)
    with pytest.raises(RuntimeError, match="group"):
        z = torch.zeros(1, 1, 512, 64, dtype=torch.int8, device=DEV)
        o = torch.ones(1, 1, 1, device=DEV)
        paged_attention_kv8(q, z, z, o, o, bt, ctx)


def test_empty_calls():
    k, v, ks, vs = C8.kv8_alloc(4, 2, 16, 64, device=DEV)
    bt = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    none = dev32(np.zeros(0, np.int32))
    q = torch.zeros(0, 4, 64, dtype=BF, device=DEV)
    assert paged_attention_kv8(q, k, v, ks, vs, bt, none).shape == q.shape
    C8.kv8_cache_write(q[:, :2], q[:, :2], k, v, ks, vs, bt, none)
    rk, _ = C8.kv8_cache_read(k, v, ks, vs, bt, dev32([0]), 0)
    assert rk.shape == (0, 2, 64)
    kept, lens = C8.kv8_cache_evict(k, v, ks, vs, bt, none, torch.zeros(0, 2, 48, device=DEV), 8, 2)
    assert kept.shape == (0, 2, 8) and lens.shape == (0,)
    # a table without pages: nothing to see
    bt = torch.zeros(2, 0, dtype=torch.int32, device=DEV)
    q = torch.ones(2, 4, 64, dtype=BF, device=DEV)
    out, lse = paged_attention_kv8(q, k, v, ks, vs, bt, dev32([5, 0]), return_lse=True)
    assert not out.float().any() and torch.isinf(lse).all()
