"""Drafted trees' attention at the end of what a table holds."""
import pytest
import torch

import plain
from test_gpu_tree import DEV, REL, build, trees
from winnow_b200 import _lib, packed_attention as pa
from winnow_b200.packed_attention_cuda import tree_decode_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("over", [3, 6, 20, 200])
def test_trees_that_reach_past_the_table(dtype, over):
    """A length the table has no room for is reported, and what it has room for stays where it is: history before
    the tree, the tree's first tokens (all of them see token 0).  `over` 20, 200: not even all of the history."""
    S, W, Q, D = 16, 5, 8, 128
    kv = build([W * S + over, 50], 2, D, S, 4, 4)
    short = pa.PackedKV(kv.k_pages, kv.k_norms, kv.v_pages, kv.v_norms, kv.page_table[:, :W], kv.seq_lens, kv.k_quant,
                        kv.v_quant, D)
    seen = trees(2, Q, 2)
    q = torch.randn(2, 8, Q, D, generator=torch.Generator().manual_seed(1)).to(DEV, dtype)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = tree_decode_attention(q, short, plain.words(seen).to(DEV), D ** -0.5, check_page_ids=False, status=status)
    assert int(status) == _lib.STATUS_BAD_POSITION
    # in 64 bits over the tokens that there are: the values past the table with nobody who sees them
    k, v = (plain.dequantised(p, n, t, short.page_table[0], W * S, S, D)
            for p, n, t in ((kv.k_pages, kv.k_norms, kv.k_quant), (kv.v_pages, kv.v_norms, kv.v_quant)))
    hist = W * S + over - Q
    allowed = torch.ones(Q, W * S, dtype=torch.bool)
    if hist < W * S:
        allowed[:, hist:] = seen[0][:, :W * S - hist]
    for h in range(8):
        s = (q[0, h].double() @ k[h // 4].T * D ** -0.5).masked_fill(~allowed.to(DEV), -torch.inf)
        want = torch.softmax(s, -1) @ v[h // 4]
        assert (got[0, h].double() - want).norm() <= REL[dtype] * want.norm()
    whole = plain.tree_attention(q[1:], pa.PackedKV(kv.k_pages, kv.k_norms, kv.v_pages, kv.v_norms, kv.page_table[1:],
                                                    kv.seq_lens[1:], kv.k_quant, kv.v_quant, D), seen[1:], D ** -0.5)
    assert (got[1:].double() - whole).norm() <= REL[dtype] * whole.norm()
