"""Drafted trees' attention where a warp's query rows differ: some do not exist, some are padding, some go another way."""
import pytest
import torch

import plain
from test_gpu_tree import DEV, REL, build, check, trees
from winnow_b200.packed_attention_cuda import tree_decode_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Q", [(1, 1), (3, 11), (6, 22), (14, 19)])
def test_rows_of_a_warp_that_do_not_exist(dtype, Hq, Q):
    kv = build([70, 600, 64], 1, 128, 16, 4, 6)
    check(kv, 3, Hq, Q, dtype, padded=Q // 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_single_rows_beyond_fp16(dtype):
    """One query of a warp too large for fp16 parts: its scores come from the codes, the other rows keep their bits."""
    kv = build([900, 75], 2, 128, 16, 4, 4)
    seen = trees(2, 6, 3)
    mask = plain.words(seen).to(DEV)
    q = torch.randn(2, 8, 6, 128, generator=torch.Generator().manual_seed(5)).to(DEV, torch.bfloat16)
    scale = 4.0
    clean = tree_decode_attention(q.to(dtype), kv, mask, scale)
    q[0, 3, 2] *= 2.0 ** 13                              # (times the scale: beyond 65 504)
    q[1, 0, 5] *= 2.0 ** 13
    q = q.to(dtype)
    got = tree_decode_attention(q, kv, mask, scale)
    want = plain.tree_attention(q, kv, seen, scale)
    for at in ((0, 3, 2), (1, 0, 5)):
        assert (got[at].double() - want[at]).norm() <= REL[dtype] * want[at].norm()
        got[at] = clean[at]
    assert torch.equal(got, clean)
