"""Attention over the 8-bit cache from several host threads on one stream (GPU)."""

import threading

import pytest
import torch

import kv8_cases as KC
from paged_attention_kv8 import paged_attention_kv8
from test_gpu_kv8 import dev32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("path", [0, 1])
def test_threads_on_one_stream(path):
    """Calls of different sizes, with and without weights, give each thread what it gets alone, bit for bit."""
    import _tak_b200 as T
    jobs = []
    for i, (seqs, Lq, ctx) in enumerate([(4, 1, [900, 1, 450, 899]), (2, 4, [300, 77]), (3, 2, [64, 800, 5])]):
        c = KC.make(("threads", i), seqs, 2, 32, 16, 128, "int8", max(ctx))
        q = torch.randn(seqs, Lq, 16, 128, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(DEV)
        jobs.append((q, KC.to_device(c), dev32(ctx), torch.zeros(seqs, 2, c.table.shape[1] * 32, device=DEV)))

    def call(job):
        q, d, ctx, weights = job
        w = torch.zeros_like(weights)
        out, lse = paged_attention_kv8(q, *d, ctx, weights=w, return_lse=True)
        return out, lse, w

    old = T.set_kernel_path(path)
    try:
        want = [call(j) for j in jobs]
        torch.cuda.synchronize()
        got = {}

        def work(i):
            torch.cuda.set_device(0)
            got[i] = [call(jobs[i]) for _ in range(60)]

        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
    finally:
        T.set_kernel_path(old)
    for i in range(len(jobs)):
        assert len(got[i]) == 60
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], r))
