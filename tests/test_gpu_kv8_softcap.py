"""Caps of the attention scores at the ends of fp32 (GPU)."""

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


@pytest.mark.parametrize("path", [0, 1])
@pytest.mark.parametrize("rows", [1, 16])
@pytest.mark.parametrize("cap", [1e20, 1e30, 8e37, 2.0 ** 126, 1e38, 2.4e38, 3.4e38, 1e39, 1e300, float("inf")])
def test_large_caps_cap_nothing(cap, rows, path):
    c = KC.make("cap", 2, 2, 32, 16, 128, "int8", 400)
    d = KC.to_device(c)
    ctx = [400, 70]
    q = torch.randn(2, 1, 2 * rows, 128, generator=torch.Generator().manual_seed(3)).to(BF)
    weights = torch.zeros(2, 2, c.table.shape[1] * 32, device=DEV)
    old = T.set_kernel_path(path)
    try:
        out, lse = paged_attention_kv8(q.to(DEV), *d, dev32(ctx), softcap=cap, weights=weights, return_lse=True)
        plain, plain_lse = paged_attention_kv8(q.to(DEV), *d, dev32(ctx), return_lse=True)
    finally:
        T.set_kernel_path(old)
    want = c.attend(q.double().numpy(), ctx)
    KC.check_attention((KC.numbers(out).astype(np.float64), lse.cpu().double().numpy(),
                        weights.cpu().double().numpy()), want, BF, 128, 2.0 ** -11)
    if cap > 2.0 ** 126:
        assert torch.equal(out, plain) and torch.equal(lse, plain_lse)


def test_caps_below_fp32s_normal_numbers_are_refused():
    c = KC.make("cap", 1, 1, 32, 16, 128, "int8", 40)
    d = KC.to_device(c)
    q = torch.ones(1, 4, 128, dtype=BF, device=DEV)
    for cap in (1e-39, 1e-45, 1e-60, float("nan"), -1e-60, -float("inf")):
        with pytest.raises((AssertionError, RuntimeError), match="softcap"):
            paged_attention_kv8(q, *d, dev32([40]), softcap=cap)
    out = paged_attention_kv8(q, *d, dev32([40]), softcap=2.0 ** -126).float().cpu()
    even = torch.from_numpy(c.values(1, 0, 0, 40).mean(0)).float()  # all scores 0 to within the cap
    mass = torch.from_numpy(np.abs(c.values(1, 0, 0, 40)).mean(0)).float()
    assert ((out[0] - even).abs() <= KC.ULP[BF] * even.abs() * 1.001 + 2.0 ** -10 * mass).all()
