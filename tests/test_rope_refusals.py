"""Calls of `qk_norm_rope` that could not give what they promise: refused before anything is launched."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from winnow_b200.rotary import qk_norm_rope


def _empty(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("shape,stretched", [((1, 8, 3, 64), "batch"), ((2, 1, 3, 64), "head"), ((2, 8, 1, 64), "token")])
def test_results_in_broadcast_tensors(shape, stretched):
    """In place they would be turned once for every copy, and elsewhere written by several blocks."""
    with FakeTensorMode():
        q, k = _empty(*shape).expand(2, 8, 3, 64), _empty(2, 2, 3, 64)
        positions, table = _empty(2, 3, dtype=torch.int32), _empty(9, 64, dtype=torch.float32)
        for into in (q, _empty(*shape).expand(2, 8, 3, 64)):
            with pytest.raises(ValueError, match="overlap themselves"):
                qk_norm_rope(q, k, positions, table, out=(into, _empty(2, 2, 3, 64)))


def test_results_in_windows_that_meet():
    with FakeTensorMode():
        windows = _empty(400).as_strided((2, 8, 3, 64), (1, 8, 2, 1))
        with pytest.raises(ValueError, match="overlap themselves"):
            qk_norm_rope(_empty(2, 8, 3, 64), _empty(2, 2, 3, 64), _empty(2, 3, dtype=torch.int32),
                         _empty(9, 64, dtype=torch.float32), out=(windows, _empty(2, 2, 3, 64)))
