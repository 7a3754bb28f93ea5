"""Calls of `qk_norm_rope` that could not give what they promise: refused before anything is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

from winnow_b200 import packed_attention as pa
from winnow_b200.packed_attention_cuda import tree_decode_attention
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


def _tangents(device):
    x, i = torch.zeros(1, 2, 3, 16, device=device), torch.zeros(1, 3, dtype=torch.int32, device=device)
    w = torch.ones(16, device=device)
    t = torch.zeros(4, 16, device=device)
    with fwAD.dual_level(), torch.no_grad():
        for args, kw in (((fwAD.make_dual(x, x), x), {}), ((x, fwAD.make_dual(x, x)), {}),
                         ((x, x), dict(v=fwAD.make_dual(x, x))), ((x, x), dict(q_weight=fwAD.make_dual(w, w)))):
            with pytest.raises(RuntimeError, match="tangents"):
                qk_norm_rope(*args, i, t, **kw)
        with pytest.raises(RuntimeError, match="tangents"):
            qk_norm_rope(x, x, i, fwAD.make_dual(t, t))
        q = pa.Quantizer(torch.eye(16, device=device), torch.zeros(16, device=device), 4)
        pages = torch.zeros(4, 2, 16, 8, dtype=torch.uint8, device=device)
        norms = torch.zeros(4, 2, 16, dtype=torch.float16, device=device)
        kv = pa.PackedKV(pages, norms, pages, norms, i, i[0, :1] + 3, q, q, 16)
        for check in (False, True):
            with pytest.raises(RuntimeError, match="tangents"):
                tree_decode_attention(fwAD.make_dual(x, x), kv, torch.zeros(1, 3, 1, dtype=torch.int32, device=device), 1.0,
                                      check_page_ids=check)


def test_tangents_are_not_dropped():
    _tangents("cpu")


@pytest.mark.gpu
def test_tangents_are_not_dropped_by_the_native_host():
    _tangents("cuda")
