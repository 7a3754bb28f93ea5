"""Buffers beside the operands of a drafted step's calls: on the operands' device and in one piece, or refused."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from winnow_b200 import _lib, packed_attention as pa
from winnow_b200.block_tables import plan_tokens
from winnow_b200.packed_attention_cuda import tree_decode_attention
from winnow_b200.packed_backend import keep_tokens
from winnow_b200.rotary import qk_norm_rope


@pytest.fixture(autouse=True)
def without_the_native_host(monkeypatch):
    """It declines what is not plain, and would ask tensors without storage for their addresses first."""
    class Declines:
        tree = keep = plan = rope = staticmethod(lambda *a: None)
    monkeypatch.setattr(_lib, "host", lambda: Declines)


def _e(*shape, dtype=torch.int32, device="cuda:0"):
    return torch.empty(*shape, dtype=dtype, device=device)


def _kv():
    pages, norms = _e(4, 2, 16, 32, dtype=torch.uint8), _e(4, 2, 16, dtype=torch.float16)
    quant = pa.Quantizer(_e(64, 64, dtype=torch.float32), _e(16, dtype=torch.float32), 4)
    return pa.PackedKV(pages, norms, pages, norms, _e(2, 3), _e(2), quant, quant, 64)


def _tree(**kw):
    return tree_decode_attention(_e(2, 4, 3, 64, dtype=torch.bfloat16), _kv(), _e(2, 3, 1), 0.1, check_page_ids=False, **kw)


def _calls():
    pages, norms = _e(1, 4, 2, 16, 32, dtype=torch.uint8), _e(1, 4, 2, 16, dtype=torch.float16)
    x, t = _e(2, 4, 3, 64, dtype=torch.bfloat16), _e(9, 64, dtype=torch.float32)
    return {"tree": _tree,
            "keep": lambda **kw: keep_tokens(pages, norms, pages, norms, _e(2, 3), _e(2), _e(2, 2), _e(2), 2, **kw),
            "plan": lambda **kw: plan_tokens(_e(2), _e(2), _e(2, 4), _e(2), _e(5), _e(1), 16, 6, **kw),
            "rope": lambda **kw: qk_norm_rope(x, x, _e(2, 3), t, **kw)}


@pytest.mark.parametrize("call", ["tree", "keep", "plan", "rope"])
def test_status_words_of_another_device(call):
    with FakeTensorMode():
        with pytest.raises(_lib.BackendError, match="cuda:1"):
            _calls()[call](status=_e(1, device="cuda:1"))


def test_a_ticket_of_another_device():
    with FakeTensorMode():
        with pytest.raises(_lib.BackendError, match="cuda:1"):
            _calls()["plan"](ticket=_e(1, device="cuda:1"))


def test_workspaces_of_another_device_or_in_pieces():
    with FakeTensorMode():
        with pytest.raises(_lib.BackendError, match="cuda:1"):
            _tree(workspace=_e(1 << 20, dtype=torch.uint8, device="cuda:1"))
        for pieces in (_e(2, dtype=torch.uint8)[:1].expand(1 << 24), _e(1 << 24, dtype=torch.uint8)[::2]):
            with pytest.raises(pa.UnsupportedLayout, match="contiguous"):
                _tree(workspace=pieces)
