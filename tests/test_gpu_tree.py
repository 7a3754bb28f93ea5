"""Attention of drafted trees against its definition in 64 bits.

Tolerances, relative to the norm of the result.  fp32 queries: sums of up to a few thousand fp32 terms,
each rounded to 2^-24: below 2e-5.  16-bit queries: the result's rounding is at most 2^-9 (bf16) or
2^-12 (fp16) of it in the mean; tensor-core operands are fp16.  A score of |s| <= ~8 nats (logits here have
a deviation of at most 2) is off by sqrt(2) * 2^-12 / sqrt(D) * |q||k| <= 8e-4 in the mean, a value
by sqrt(2) * 2^-12, a probability by 2^-12, together below 1.2e-3: 4e-3 for bf16, 2e-3 for fp16.
"""
import pytest
import torch

import plain
from winnow_b200 import _lib, packed_attention as pa
from winnow_b200.cache import _get_quantizer
from winnow_b200.packed_attention_cuda import (packed_decode_attention, tree_decode_attention,
                                               tree_workspace_bytes)

pytestmark = pytest.mark.gpu
DEV = "cuda"
REL = {torch.float32: 2e-5, torch.bfloat16: 4e-3, torch.float16: 2e-3}


def build(lens, Hkv, D, S, bw_k, bw_v, seed=0, spare=3, scale_k=1.0):
    """A paged cache of random codes: page ids in random order, unused entries -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(L, 0) // S) for L in lens]
    P = sum(need) + spare
    order = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    sides = []
    for bw, sc in ((bw_k, scale_k), (bw_v, 1.0)):
        pages = torch.randint(0, 256, (P, Hkv, S, D * bw // 8), generator=g, dtype=torch.uint8)
        norms = (D ** 0.5 * sc * torch.exp(0.3 * torch.randn(P, Hkv, S, generator=g))).half()
        sides += [pages.to(DEV), norms.to(DEV)]
    kq, vq = (pa.Quantizer.from_tq(_get_quantizer(b, D, DEV, s)) for b, s in ((bw_k, 42), (bw_v, 43)))
    return pa.PackedKV(*sides, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), kq, vq, D)


def trees(B, Q, seed, padded=0):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for b in range(B):
        real = Q - (padded if b % 2 else 0)
        rows.append([-1 if i == 0 else max(0, i - 1 - int(torch.randint(0, 6, (1,), generator=g))) if i < real else -2
                     for i in range(Q)])
    return plain.reach(rows)


def check(kv, B, Hq, Q, dtype, seed=1, padded=0, mult=1.0, seen=None, rel=None, **kw):
    g = torch.Generator().manual_seed(seed)
    D = kv.head_dim
    q = (mult * torch.randn(B, Q, Hq, D, generator=g)).to(DEV, dtype).transpose(1, 2)
    seen = trees(B, Q, seed, padded) if seen is None else seen
    mask = plain.words(seen).to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = tree_decode_attention(q, kv, mask, D ** -0.5, status=status, **kw)
    want = plain.tree_attention(q, kv, seen, D ** -0.5)
    assert got.shape == (B, Hq, Q, D) and got.dtype == dtype
    assert int(status) == 0
    assert torch.isfinite(got).all()
    err = (got.double() - want).norm() / want.norm().clamp_min(1e-30)
    assert err <= (rel or REL[dtype]), f"relative L2 {err:.2e}"
    empty = ~seen.any(-1)
    assert not got.transpose(1, 2)[empty.to(DEV)].any()
    return q, mask, got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,Q,S", [
    ([1], 1, 1, 1, 16),                         # one token that sees itself
    ([5, 3], 4, 2, 3, 16),                      # no history, two tokens of history
    ([64, 65, 63, 128], 8, 2, 8, 16),           # tile borders
    ([1000], 8, 2, 8, 16),
    ([700, 33, 200, 1], 28, 4, 1, 32),          # one query token per sequence: causal decode
    ([300, 96, 100], 14, 2, 31, 64),            # 217 rows: two row blocks
    ([257, 96, 512], 16, 8, 33, 16),            # two mask words
    ([513], 32, 2, 96, 32),                     # three mask words, twelve row blocks
    ([150], 40, 2, 5, 16),                      # twenty query heads to a kv head
])
def test_head_layouts_and_lengths(dtype, lens, Hq, Hkv, Q, S):
    kv = build(lens, Hkv, 128, S, 4, 4)
    check(kv, len(lens), Hq, Q, dtype, padded=Q // 3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("widths", [(4, 4), (4, 6), (6, 6), (8, 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tensor_core_widths(D, widths, dtype):
    kv = build([777, 40, 333], 2, D, 16, *widths)
    side = [_lib.Side(p.data_ptr(), n.data_ptr(), p.stride(0), p.stride(1), n.stride(0), n.stride(1), None, None, None,
                      b) for p, n, b in ((kv.k_pages, kv.k_norms, widths[0]), (kv.v_pages, kv.v_norms, widths[1]))]
    assert _lib.lib().wtq_tree_on_tensor_cores(side[0], side[1], _lib.dtype_code(dtype), D, 16) == 1
    check(kv, 3, 14, 17, dtype)


@pytest.mark.parametrize("D,widths,S", [(128, (2, 3), 16), (96, (5, 5), 16), (64, (3, 8), 7), (256, (4, 4), 32),
                                        (16, (4, 4), 1), (80, (6, 2), 5), (128, (4, 4), 24), (200, (8, 4), 16),
                                        (4, (2, 4), 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_of_the_fp32_scan(D, widths, S, dtype):
    kv = build([130, 17, 260], 2, D, S, *widths)
    check(kv, 3, 6, 9, dtype, padded=2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mixed_lengths_and_empty_sequences(dtype):
    lens = [0, 4000, 9, 0, 0, 1500, 70, 2, 0]    # 2: shorter than the tree; 0: nothing stored
    kv = build(lens, 2, 128, 16, 4, 4)
    check(kv, len(lens), 8, 9, dtype, padded=4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_one_long_history_among_short_ones(dtype):
    kv = build([30000, 40, 12, 300], 2, 128, 64, 4, 4)
    check(kv, 4, 8, 16, dtype)


def test_masks_that_leave_everything_out():
    kv = build([40, 500], 2, 128, 16, 4, 4)
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.full((2, 8, 5, 128), float("nan"), dtype=dtype, device=DEV)
        out = tree_decode_attention(q, kv, torch.zeros(2, 5, 1, dtype=torch.int32, device=DEV), 0.1)
        assert not out.any() and not out.isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nan_queries_of_padding_reach_nobody(dtype):
    kv = build([200, 90], 2, 128, 16, 4, 4)
    seen = trees(2, 6, 3, padded=2)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 8, 6, 128, generator=g).to(DEV, dtype)
    mask = plain.words(seen).to(DEV)
    clean = tree_decode_attention(q, kv, mask, 0.09)
    q[1, :, 4:] = float("nan")
    dirty = tree_decode_attention(q, kv, mask, 0.09)
    assert torch.equal(clean, dirty)


@pytest.mark.parametrize("lens", [[200, 90], [9000, 90]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_query_that_is_not_a_number_spoils_its_own_row(dtype, lens):
    kv = build(lens, 2, 128, 16, 4, 4)
    mask = plain.words(trees(2, 6, 3)).to(DEV)
    q = torch.randn(2, 8, 6, 128, generator=torch.Generator().manual_seed(5)).to(DEV, dtype)
    clean = tree_decode_attention(q, kv, mask, 0.09)
    q[0, 3, 2, 7] = float("nan")
    q[1, 0, 0] = float("nan")
    dirty = tree_decode_attention(q, kv, mask, 0.09)
    assert dirty[0, 3, 2].isnan().all() and dirty[1, 0, 0].isnan().all()
    dirty[0, 3, 2], dirty[1, 0, 0] = clean[0, 3, 2], clean[1, 0, 0]
    assert torch.equal(clean, dirty)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_queries_beyond_fp16(dtype):
    """|q| of 1e6: logits of 1e5 and more, all weight on one token, whose value comes back as it is stored
    (fp16 centroid times norm: 2^-11 each at most)."""
    kv = build([300, 40], 2, 128, 16, 4, 4)
    check(kv, 2, 8, 5, dtype, mult=1e6, rel=1e-3 + (4e-3 if dtype == torch.bfloat16 else 0))


def test_bits_past_the_tree_are_ignored():
    kv = build([200], 2, 128, 16, 4, 4)
    seen = trees(1, 5, 3)
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.randn(1, 8, 5, 128, generator=g).to(DEV, dtype)
        mask = plain.words(seen).to(DEV)
        assert torch.equal(tree_decode_attention(q, kv, mask, 0.09),
                           tree_decode_attention(q, kv, mask | ~0x1f, 0.09))


@pytest.mark.parametrize("mult", [8.0, 40.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_large_logits(mult, dtype):
    """Logits of tens of nats (deviation 8, 40).  16-bit scores near the maximum are re-scored in fp32 beyond 16.6 nats,
    whose codes carry no rounding: the bound of the ordinary case holds.  fp32: a score of |s| <= 200 nats is off by
    200 * 2^-24 * ~8 = 1e-4 at most."""
    kv = build([400, 130], 2, 128, 16, 4, 4)
    check(kv, 2, 8, 6, dtype, mult=mult, rel=1.5e-4 if dtype == torch.float32 else None)


def test_chain_is_causal_attention():
    """A chain of drafts is a causal chunk: token i as one-token decode over the first hist + i + 1 tokens."""
    kv = build([300, 81], 2, 128, 16, 4, 4)
    Q = 7
    seen = torch.ones(Q, Q, dtype=torch.bool).tril().expand(2, Q, Q)
    for dtype in (torch.float32, torch.bfloat16):
        q, _, got = check(kv, 2, 8, Q, dtype, seen=seen)
        for i in range(Q):
            view = pa.PackedKV(kv.k_pages, kv.k_norms, kv.v_pages, kv.v_norms, kv.page_table,
                               kv.seq_lens - (Q - 1 - i), kv.k_quant, kv.v_quant, 128)
            one = packed_decode_attention(q[:, :, i:i + 1].contiguous(), view, 128 ** -0.5)
            assert (got[:, :, i:i + 1].float() - one.float()).norm() <= 8e-3 * one.float().norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Queries and results as slices of wider buffers, a strided table and mask, pages of one layer of a pool."""
    kv = build([333, 64, 90], 4, 128, 16, 4, 6)
    B, Hq, Q, D = 3, 8, 6, 128
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(B, Q, Hq + 3, D + 8, generator=g).to(DEV, dtype)
    q = wide[:, :, 2:2 + Hq, 8:].transpose(1, 2)
    seen = trees(B, Q, 1, padded=1)
    mask = torch.zeros(B, Q + 2, 3, dtype=torch.int32, device=DEV)[:, 1:1 + Q, 1:2]
    mask.copy_(plain.words(seen))
    table = torch.full((B, kv.page_table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)[:, :kv.page_table.shape[1]]
    table.copy_(kv.page_table)
    pool = [torch.stack([t, t.flip(0)], 1) for t in (kv.k_pages, kv.k_norms, kv.v_pages, kv.v_norms)]
    view = pa.PackedKV(pool[0][:, 0], pool[1][:, 0], pool[2][:, 0], pool[3][:, 0], table, kv.seq_lens, kv.k_quant,
                       kv.v_quant, D)
    want = tree_decode_attention(q.contiguous(), kv, mask.contiguous(), 0.09)
    room = torch.full((B, Hq + 2, Q + 1, D + 8), 7.0, dtype=dtype, device=DEV)
    out = room[:, 1:1 + Hq, :Q, :D]
    assert tree_decode_attention(q, view, mask, 0.09, out=out, check_page_ids=False) is out
    assert torch.equal(out, want)
    assert (room[:, 0] == 7).all() and (room[:, -1] == 7).all() and (room[:, :, -1] == 7).all() \
        and (room[..., D:] == 7).all()
    assert torch.equal(tree_decode_attention(q, view, mask, 0.09, check_page_ids=False), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_outside_the_pool(dtype):
    kv = build([120, 100], 2, 128, 16, 4, 4)
    kv.page_table[0, 2] = 10 ** 6
    kv.page_table[1, 0] = -7
    seen = trees(2, 4, 1)
    q = torch.randn(2, 8, 4, 128, device=DEV).to(dtype)
    mask = plain.words(seen).to(DEV)
    with pytest.raises(pa.UnsupportedLayout):
        tree_decode_attention(q, kv, mask, 0.09)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = tree_decode_attention(q, kv, mask, 0.09, check_page_ids=False, status=status)
    assert int(status) == _lib.STATUS_BAD_PAGE
    want = plain.tree_attention(q, kv, seen, 0.09)           # rows of such pages read as zeros
    assert (got.double() - want).norm() <= REL[dtype] * want.norm()


def test_the_same_call_twice_and_on_another_stream():
    kv = build([900, 350, 40], 4, 128, 16, 4, 4)
    for dtype in (torch.float32, torch.bfloat16):
        q, mask, first = check(kv, 3, 16, 12, dtype)
        assert torch.equal(first, tree_decode_attention(q, kv, mask, 128 ** -0.5, check_page_ids=False))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [tree_decode_attention(q, kv, mask, 128 ** -0.5, check_page_ids=False) for _ in range(3)]
        here = [tree_decode_attention(q, kv, mask, 128 ** -0.5, check_page_ids=False) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(first, x) for x in other + here)


def test_captured_and_replayed():
    kv = build([900, 350], 4, 128, 16, 4, 4)
    for dtype in (torch.float32, torch.bfloat16):
        q, mask, first = check(kv, 2, 16, 12, dtype)
        ws = torch.empty(tree_workspace_bytes(2, 16, 4, 12, 128, DEV), dtype=torch.uint8, device=DEV)
        out = torch.zeros_like(first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tree_decode_attention(q, kv, mask, 128 ** -0.5, check_page_ids=False, out=out, workspace=ws)
        ws.fill_(255)                                        # (needs no preparation)
        graph.replay()
        assert torch.equal(out, first)
        kv.seq_lens.sub_(5)                                  # shorter histories, the same graph
        q.mul_(0.5)
        graph.replay()
        assert torch.equal(out, tree_decode_attention(q, kv, mask, 128 ** -0.5, check_page_ids=False))
        kv.seq_lens.add_(5)


def test_more_sequences_than_a_launch_takes():
    B = 2050
    kv = build([20] * B, 1, 64, 16, 4, 4)
    check(kv, B, 2, 2, torch.bfloat16)


@pytest.mark.parametrize("dtype,widths", [(torch.float32, (4, 4)), (torch.bfloat16, (4, 4)), (torch.bfloat16, (8, 8)),
                                          (torch.bfloat16, (4, 6))])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_norms_that_are_not_numbers_reach_those_that_see_them(dtype, widths, bad):
    """Tree tokens with such norms: siblings and tokens after them keep their bits, descendants are NaN."""
    lens, Q = [200, 73, 3000], 13
    kv = build(lens, 2, 128, 16, *widths)
    seen = trees(3, Q, 5)
    q = torch.randn(3, 8, Q, 128, generator=torch.Generator().manual_seed(3)).to(DEV, dtype)
    mask = plain.words(seen).to(DEV)
    want = tree_decode_attention(q, kv, mask, 0.09)
    spoilt = torch.zeros(3, Q, dtype=torch.bool)
    for b, L in enumerate(lens):
        for j in (4, 9):
            at = L - Q + j
            page = int(kv.page_table[b, at // 16])
            kv.v_norms[page, :, at % 16] = bad
            if j == 9:
                kv.k_norms[page, :, at % 16] = bad
            spoilt[b] |= seen[b, :, j]
    assert spoilt.any() and not spoilt.all()
    got = tree_decode_attention(q, kv, mask, 0.09).transpose(1, 2)
    spoilt = spoilt.to(DEV)
    assert got[spoilt].isnan().all()
    assert torch.equal(got[~spoilt], want.transpose(1, 2)[~spoilt])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [5, 4000, 8900])
def test_a_norm_in_the_history_that_is_not_a_number_is_not_lost(dtype, at):
    """One in a long history, whose other pieces may have far larger maxima: every row sees it."""
    kv = build([9000, 90], 2, 128, 16, 4, 4)
    q = (100 * torch.randn(2, 8, 3, 128, generator=torch.Generator().manual_seed(3))).to(DEV, dtype)
    mask = plain.words(trees(2, 3, 1)).to(DEV)
    want = tree_decode_attention(q, kv, mask, 0.09)
    kv.v_norms[int(kv.page_table[0, at // 16]), 1, at % 16] = float("inf")
    got = tree_decode_attention(q, kv, mask, 0.09)
    assert got[0, 4:].isnan().all()
    assert torch.equal(got[0, :4], want[0, :4]) and torch.equal(got[1], want[1])
