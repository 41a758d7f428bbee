"""The 8-bit KV cache at the sizes where its kernels change form (GPU): long
selections, windows over clusters, many query rows, caches past 2^31 codes."""

import numpy as np
import pytest
import torch

import _tak_b200 as T
import kv8_cache as C8
import kv8_cases as KC
from paged_attention_kv8 import paged_attention_kv8
from test_gpu_kv8 import check_rot, dev32, rot_inputs
from rotary_nd import rotary_nd

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("rows,budget,recent", [(5000, 4500, 10), (20000, 9000, 3000), (70000, 600, 0),
                                                (131072, 700, 700), (140001, 500, 50)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_long(rows, budget, recent, ties):
    """One to sixteen CTAs per (sequence, head) in selection and moves, and a
    sequence too long for the selection in registers."""
    c = KC.make(("long", rows), 2, 1, 64, 16, 16, "int8", rows)
    d = KC.to_device(c)
    g = np.random.default_rng(rows)
    w = g.random((2, 1, c.table.shape[1] * 64)).astype(np.float32) ** 8
    if ties:
        w = np.round(w * 2).astype(np.float32)
    ctx = [rows, rows // 3]
    dw = torch.from_numpy(w.copy()).to(DEV)
    kept, lens = C8.kv8_cache_evict(*d, dev32(ctx), dw, budget, recent)
    rk, rl = c.evict(ctx, w, budget, recent)
    assert np.array_equal(lens.cpu().numpy(), rl) and np.array_equal(kept.cpu().numpy(), rk)
    assert np.array_equal(dw.cpu().numpy(), w)
    KC.same(c, d)


ATT = [  # seqs, q heads, kv heads, dim, block, group, contexts, queries
    (2, 12, 1, 256, 32, 16, [257, 30], 1),
    (2, 8, 1, 256, 64, 32, [129, 600], 3),
    (1, 4, 1, 200, 16, 16, [150], 11),
    (2, 10, 1, 64, 48, 16, [255, 5], 1),
    (3, 9, 1, 128, 128, 64, [1, 128, 500], 2),
    (1, 3, 3, 128, 16, 16, [260], 40),
    (40, 2, 1, 64, 16, 16, [(7 * i) % 120 for i in range(40)], 1),
    (1, 16, 1, 112, 32, 32, [2100], 2),
    (1, 4, 1, 208, 16, 16, [150], 11),
]


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("i", range(len(ATT)))
def test_attention_many_rows(i, dtype, code):
    seqs, H, hkv, dim, block, group, ctx, Lq = ATT[i]
    c = KC.make(("rows", i), seqs, hkv, block, group, dim, code, max(ctx))
    d = KC.to_device(c)
    q = torch.randn(seqs, Lq, H, dim, generator=torch.Generator().manual_seed(i)).to(dtype)
    weights = torch.zeros(seqs, hkv, c.table.shape[1] * block, device=DEV)
    out, lse = paged_attention_kv8(q.to(DEV), *d, dev32(ctx), weights=weights, return_lse=True)
    # rows of codes whose stride is no multiple of 16 bytes cannot be copied by TMA
    assert T.last_kernel() == ("kv8_attention_tc" if dim % 16 == 0 else "kv8_attention_generic")
    want = c.attend(q.double().numpy(), ctx)
    KC.check_attention((KC.numbers(out).astype(np.float64), lse.cpu().double().numpy(),
                        weights.cpu().double().numpy()), want, dtype, dim, 2.0 ** -11)
    assert T.read_device_error() == 0


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attention_hidden_v_scale(code):
    """A NaN V scale reaches the query rows that see a key of its tile, and no other."""
    c = KC.make("vnan", 1, 2, 16, 16, 64, code, 48)
    c.scales[1][c.table[0, 2], 0, 0] = np.nan  # keys 32 .. 47 of head 0
    d = KC.to_device(c)
    for G in (1, 4):  # four and sixteen rows a head
        q = torch.randn(1, 4, 2 * G, 64, generator=torch.Generator().manual_seed(G)).to(BF)
        out, lse = paged_attention_kv8(q.to(DEV), *d, dev32([34]), return_lse=True)
        bad = torch.isnan(out.float()).all(-1)[0].cpu()
        any_bad = torch.isnan(out.float()).any(-1)[0].cpu()
        want = torch.zeros(4, 2 * G, dtype=torch.bool)
        want[2:, :G] = True  # query i sees 31 + i keys
        assert torch.equal(bad, want) and torch.equal(any_bad, want)
        assert torch.isfinite(lse).all()  # the softmax sums do not involve V


def test_offsets_past_32_bits():
    """Pages past 2^31 codes: every operator gives what it gives on a small pool."""
    heads, block, group, dim, far = 8, 128, 16, 128, 16400
    lens = [700, 129]
    small = KC.make("far", 2, heads, block, group, dim, "int8", max(lens) + 40)
    a = KC.to_device(small)
    b = [torch.zeros(far + small.nb, heads, block, dim, dtype=torch.int8, device=DEV) for _ in range(2)]
    s = [torch.zeros(far + small.nb, heads, block // group, device=DEV) for _ in range(2)]
    assert b[0].numel() > 2 ** 31
    for w in range(2):
        b[w][far:] = a[w]
        s[w][far:] = a[2 + w]
    big = (*b, *s, a[4] + far)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(40, heads, dim, generator=g).to(BF).to(DEV) for _ in range(2))
    q = torch.randn(2, 32, dim, generator=g).to(BF).to(DEV)
    got = []
    for d in (a, big):
        C8.kv8_cache_write(k, v, *d, dev32(lens), dev32([0, 33, 40]))
        n = [lens[0] + 33, lens[1] + 7]
        rows = C8.kv8_cache_read(*d, dev32([0, n[0], n[0] + n[1]]), sum(n))
        weights = torch.zeros(2, heads, d[4].shape[1] * block, device=DEV)
        out = paged_attention_kv8(q, *d, dev32(n), weights=weights)
        kept, left = C8.kv8_cache_evict(*d, dev32(n), weights, 200, 20)
        got.append((rows[0], rows[1], out, weights, kept, left, *[t[-small.nb:].clone() for t in d[:4]]))
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_write_groups_too_large_for_registers(code):
    c = KC.make("huge", 1, 1, 256, 256, 256, code, 600)
    d = KC.to_device(c)
    x = torch.randn(300, 1, 256, generator=torch.Generator().manual_seed(8)).to(HF)
    C8.kv8_cache_write(x.to(DEV), x.to(DEV), *d, dev32([250]), dev32([0, 300]))
    for w in (0, 1):
        c.write(w, x.float().numpy(), [250], [0, 300])
    KC.same(c, d)


def test_write_many_short_sequences():
    """More sequences than one round of the search looks at, empty ones among them."""
    n = 300
    counts = [(i * 7) % 5 for i in range(n)]
    starts = [(i * 11) % 33 for i in range(n)]
    c = KC.make("many", n, 1, 16, 16, 64, "int8", 40)
    d = KC.to_device(c)
    cu = np.concatenate([[0], np.cumsum(counts)])
    x = torch.randn(int(cu[-1]), 1, 64, generator=torch.Generator().manual_seed(8)).to(BF)
    C8.kv8_cache_write(x.to(DEV), x.to(DEV), *d, dev32(starts), dev32(cu))
    for w in (0, 1):
        c.write(w, x.float().numpy(), starts, cu)
    KC.same(c, d)
    lens = [a + b for a, b in zip(starts, counts)]
    cr = np.concatenate([[0], np.cumsum(lens)])
    k, _ = C8.kv8_cache_read(*d, dev32(cr), int(cr[-1]), dtype=FF)
    for s in range(0, n, 17):
        assert np.array_equal(KC.numbers(k)[cr[s]:cr[s + 1], 0], c.values(0, s, 0, lens[s]).astype(np.float32))


@pytest.mark.parametrize("dtype", [BF, FF])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,axes", [(2500, 3, 1, 64, 64, 2), (3, 2, 1, 1024, 1024, 1),
                                                          (2400, 1, 1, 256, 192, 3), (5, 70, 0, 64, 32, 2)])
def test_rotary_sizes(dtype, il, tokens, heads, kv, dim, rot, axes):
    q, k, pos, inv, sec = rot_inputs(tokens, tokens, heads, max(kv, 1), dim, rot, axes, dtype)
    qo, ko = rotary_nd(q.to(DEV), k.to(DEV) if kv else None, pos.to(DEV), inv.to(DEV), sec, interleaved=il)
    check_rot(qo, q, pos, inv, sec, il, False)
    if kv:
        check_rot(ko, k, pos, inv, sec, il, False)


@pytest.mark.parametrize("dim", [64, 72])
def test_write_ends_with_its_rows(dim):
    """A cu_seqlens that runs past the rows of k and v writes those that there are."""
    c = KC.make("past", 2, 2, 32, 16, dim, "int8", 120)
    d = KC.to_device(c)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(60, 2, dim, generator=g).to(BF) for _ in range(2))
    C8.kv8_cache_write(k.to(DEV), v.to(DEV), *d, dev32([3, 5]), dev32([0, 41, 90]))
    for w, x in enumerate((k, v)):
        c.write(w, x.float().numpy(), [3, 5], [0, 41, 60])
    KC.same(c, d)


def test_graph_keeps_its_scratch():
    """A captured call replays right after calls on its stream that needed more
    scratch, and after the memory that they gave back was overwritten."""
    c = KC.make("graph", 4, 2, 64, 16, 128, "int8", 900)
    d = KC.to_device(c)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to("cuda")
    ctx = torch.tensor([900, 1, 450, 899], dtype=torch.int32, device="cuda")
    many = torch.randn(4, 600, 8, 128, device="cuda").to(torch.bfloat16)
    weights = torch.zeros(4, 2, 960, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        want = paged_attention_kv8(q, *d, ctx)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            got = paged_attention_kv8(q, *d, ctx)
        paged_attention_kv8(many, *d, ctx, weights=weights)
        keep = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
        got.zero_()
        g.replay()
    st.synchronize()
    assert torch.equal(want, got)
    assert all(bool((x == 255).all()) for x in keep)


def test_large_scratch_is_not_kept(monkeypatch):
    """Scratch above the limit is taken from the allocator for the call alone, with the same results."""
    import paged_attention_kv8 as A
    c = KC.make("scratch", 3, 2, 32, 16, 128, "int8", 700)
    d = KC.to_device(c)
    q = torch.randn(3, 40, 16, 128, generator=torch.Generator().manual_seed(5)).to(BF).to(DEV)
    ctx = dev32([700, 44, 333])
    w1, w2 = (torch.zeros(3, 2, 704, device=DEV) for _ in range(2))
    a = paged_attention_kv8(q, *d, ctx, weights=w1)
    monkeypatch.setattr(A, "_KEEP", 1 << 16)
    monkeypatch.setattr(T, "_ws", {})
    b = paged_attention_kv8(q, *d, ctx, weights=w2)
    assert torch.equal(a, b) and torch.equal(w1, w2)
    assert all(x.numel() <= 1 << 20 for x in T._ws.values())
