"""Drafted trees' attention where runs are made of pieces of one tile and of several by turns: a stream that has no
tile in a piece must leave the state of the piece before alone until it has been read."""
import pytest
import torch

from test_gpu_tree import build, check
from winnow_b200.packed_attention_cuda import tree_decode_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("widths", [(4, 4), (4, 6), (8, 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_pieces_of_one_tile_after_pieces_of_two(dtype, widths):
    # 148 and more sequences a wave, a block's run a few tiles: 128 tokens (two tiles), then 40 (one), over and over
    lens = [128, 40, 100, 64, 65, 9] * 60
    kv = build(lens, 2, 128, 16, *widths)
    q, mask, first = check(kv, len(lens), 8, 5, dtype)
    for _ in range(20):
        assert torch.equal(first, tree_decode_attention(q, kv, mask, 128 ** -0.5, check_page_ids=False))


def test_runs_that_end_one_tile_into_a_group():
    """Row blocks of a long history: every run boundary leaves a piece, of one tile among others."""
    for L in (64 * 37 + 5, 64 * 75 + 1):
        kv = build([L, 64, L - 700], 4, 64, 16, 6, 6)
        q, mask, first = check(kv, 3, 32, 40, torch.float16)
        for _ in range(5):
            assert torch.equal(first, tree_decode_attention(q, kv, mask, 64 ** -0.5, check_page_ids=False))
