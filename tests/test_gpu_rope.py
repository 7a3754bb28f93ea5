"""Norms with the position rotation against their definition in 64 bits.

Tolerance of an element: its rounding, eps / 2 of its value; and fp32 arithmetic on the row: the norm is
off by (D / 32 + 8) * 2^-24 relative (a thread's share summed in order, then a tree of five), products and
the rotation by 5 * 2^-24 of |a| + |b|, with D <= 256 below 32 * 2^-24 = 2e-6 of the pair's size."""
import pytest
import torch

import plain
from winnow_b200 import _lib
from winnow_b200.rotary import qk_norm_rope, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda"


def assert_close(got, x, positions, table, weight, eps, interleaved):
    want = plain.norm_rope(x, positions, table, weight, eps, interleaved)
    y = plain.norm_rope(x, positions, table, weight, eps, interleaved, turned=False)
    size = want.abs() + 2e-6 / (torch.finfo(x.dtype).eps / 2) * y.abs().amax(-1, keepdim=True)
    bad = (got.double() - want).abs() > torch.finfo(x.dtype).eps / 2 * size * (1 + 1e-3) + 1e-7 * (x.dtype == torch.float16)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"


def inputs(B, n, Hq, Hkv, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, n, Hq + 2 * Hkv, D, generator=g).to(DEV, dtype)
    cut = [qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]]
    return [t.transpose(1, 2) for t in cut], g


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,n,Hq,Hkv,D,rot", [(1, 1, 14, 2, 64, 64), (3, 5, 8, 2, 128, 128), (2, 7, 4, 4, 96, 48),
                                              (1, 300, 32, 8, 128, 64), (2, 3, 3, 1, 256, 256), (1, 4, 2, 1, 16, 16),
                                              (2, 2, 5, 5, 80, 20), (1, 3, 2, 1, 10, 6), (1, 2, 2, 2, 7, 2),
                                              (40, 33, 28, 4, 128, 128), (1, 2, 1, 1, 250, 250)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("interleaved", [True, False])
def test_against_the_definition(dtype, B, n, Hq, Hkv, D, rot, norm, interleaved):
    (q, k, v), g = inputs(B, n, Hq, Hkv, D, dtype)
    table = rotary_table(rot, 500, base=1e6)
    positions = torch.randint(-1, 500, (B, n), generator=g, dtype=torch.int32).to(DEV)
    ws = [(1 + 0.3 * torch.randn(D, generator=g)).to(DEV, dtype) if norm else None for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    qo, ko = qk_norm_rope(q, k, positions, table, q_weight=ws[0], k_weight=ws[1], interleaved=interleaved, status=status)
    assert_close(qo, q, positions, table, ws[0], 1e-6, interleaved)
    assert_close(ko, k, positions, table, ws[1], 1e-6, interleaved)
    assert int(status) == 0 and qo.shape == q.shape and qo.dtype == dtype
    out3 = qk_norm_rope(q, k, positions, table, q_weight=ws[0], k_weight=ws[1], interleaved=interleaved, v=v)
    assert torch.equal(out3[0], qo) and torch.equal(out3[1], ko) and torch.equal(out3[2], v)


def test_far_positions_keep_their_angles():
    t = rotary_table(128, 1 << 17)
    p = 131071
    freq = 10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    want = torch.cat([(p * freq).cos(), (p * freq).sin()])
    assert (t[p].double().cpu() - want).abs().max() < 1e-7


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [128, 30])
def test_in_place_in_the_projection(dtype, D):
    (q, k, v), g = inputs(3, 6, 8, 2, D, dtype)
    table = rotary_table(D // 2 // 2 * 2, 64)
    positions = torch.randint(0, 64, (3, 6), generator=g, dtype=torch.int32).to(DEV)
    w = torch.ones(D, device=DEV, dtype=dtype)
    want = qk_norm_rope(q, k, positions, table, q_weight=w, k_weight=w)
    kept = v.clone()
    got = qk_norm_rope(q, k, positions, table, q_weight=w, k_weight=w, out=(q, k))
    assert got[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)


def test_into_given_tensors_and_mixed_weights():
    (q, k, v), g = inputs(2, 1, 8, 2, 128, torch.bfloat16)
    table = rotary_table(128, 64)
    positions = torch.tensor([[3], [60]], dtype=torch.int32, device=DEV)
    w = (1 + torch.rand(128, generator=g)).to(DEV)           # fp32 weights beside bf16 rows
    out = [torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in (q, k, v)]
    qk_norm_rope(q, k, positions, table, k_weight=w, v=v, out=out)
    assert_close(out[0], q, positions, table, None, 1e-6, False)
    assert_close(out[1], k, positions, table, w, 1e-6, False)
    assert torch.equal(out[2], v)


def test_padding_and_positions_past_the_table():
    (q, k, _), _ = inputs(2, 3, 4, 2, 128, torch.bfloat16)
    q[0, :, 1] = float("nan")
    k[0, :, 1] = float("inf")
    table = rotary_table(128, 10)
    positions = torch.tensor([[2, -1, 9], [10, 0, -5]], dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    w = torch.ones(128, device=DEV, dtype=torch.bfloat16)
    qo, ko = qk_norm_rope(q, k, positions, table, q_weight=w, k_weight=w, status=status)
    assert int(status) == _lib.STATUS_BAD_POSITION
    gone = torch.tensor([[False, True, False], [True, False, True]], device=DEV)
    for t in (qo, ko):
        assert not t.transpose(1, 2)[gone].any() and t.isfinite().all() and t.transpose(1, 2)[~gone].any()


@pytest.mark.parametrize("offset", [0, 1])
def test_odd_strides(offset):
    """Rows off 16-byte borders, tokens and heads transposed, positions and table in wider buffers."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(2, 6, 5, 128 + 9, generator=g).to(DEV, torch.bfloat16)
    q, k = wide[:, :4, :, offset:offset + 128], wide[:, 4:, :, offset:offset + 128]
    table = torch.zeros(50, 140, device=DEV)[:, 3:131]
    table.copy_(rotary_table(128, 50))
    positions = torch.randint(0, 50, (2, 9), generator=g, dtype=torch.int32).to(DEV)[:, 2:7]
    qo, ko = qk_norm_rope(q, k, positions, table)
    assert_close(qo, q, positions, table, None, 1e-6, False)
    assert_close(ko, k, positions, table, None, 1e-6, False)


def test_captured():
    (q, k, _), _ = inputs(2, 4, 8, 2, 128, torch.bfloat16)
    table, positions = rotary_table(128, 99), torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    out = [torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in (q, k)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qk_norm_rope(q, k, positions, table, out=out)
    positions.copy_(torch.arange(8).view(2, 4) * 12)
    graph.replay()
    want = qk_norm_rope(q, k, positions, table)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
