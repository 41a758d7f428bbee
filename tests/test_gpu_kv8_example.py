"""The serving example runs, with both code types."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_serving_example(codes):
    spec = importlib.util.spec_from_file_location(
        "kv8_serving", os.path.join(HERE, "triton-ascend-kernels_b200", "examples", "kv8_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    r = m.main(codes=codes, verbose=False)
    # rows N(0, 1): an element is off by at most half a step, 4.5 sigma / 254 (int8) or 2^-4 of itself
    # (e4m3), in K (through the scores) and in V alike
    assert 0 < r["worst"] < (0.05 if codes == torch.int8 else 0.2)
    assert r["evictions"] >= 1 and int(r["contexts"].max()) <= 720
    assert torch.isfinite(r["answer"].float()).all() and r["answer"].shape == (100, 32, 128)
    assert torch.isfinite(r["weights"]).all()
