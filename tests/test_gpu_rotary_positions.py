"""Types of the rotary positions (GPU)."""

import pytest
import torch

from rotary_nd import rotary_nd
from test_gpu_kv8 import check_rot, rot_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_fractional_positions_are_refused():
    q, k, pos, inv, sec = rot_inputs(1, 9, 2, 1, 64, 64, 2, torch.float32)
    for t in (torch.float32, torch.float64, torch.bfloat16):
        with pytest.raises(AssertionError, match="integers"):
            rotary_nd(q.to(DEV), k.to(DEV), (pos.to(t) / 4).to(DEV), inv.to(DEV), sec)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.uint8])
def test_integer_positions_of_other_widths(dtype):
    q, k, pos, inv, sec = rot_inputs(2, 9, 2, 1, 64, 64, 2, torch.float32, high=100)
    qo, ko = rotary_nd(q.to(DEV), k.to(DEV), pos.to(dtype).to(DEV), inv.to(DEV), sec)
    check_rot(qo, q, pos, inv, sec, False, False)
    check_rot(ko, k, pos, inv, sec, False, False)
