"""Drafted trees' attention where a few tokens carry a row: the rounding of their probabilities to 16 bits cancels
between the value sum and its denominator."""
import math

import pytest
import torch

import plain
from winnow_b200 import packed_attention as pa
from winnow_b200.cache import _get_quantizer
from winnow_b200.packed_attention_cuda import tree_decode_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("widths", [(4, 4), (4, 6), (8, 8)])
@pytest.mark.parametrize("lead", [5.1, 5.3, 5.55, 6.8, 7.4])
def test_two_tokens_carry_the_rows(widths, lead):
    D, S, H, Q, L, first, second = 128, 16, 2, 8, 208, 3, 130
    # (as many groups of one sequence and kv head as multiprocessors: each is a run, with one reference a stream)
    B = torch.cuda.get_device_properties(DEV).multi_processor_count // H
    g = torch.Generator().manual_seed(int(10 * lead))
    kq, vq = _get_quantizer(widths[0], D, DEV, 42), _get_quantizer(widths[1], D, DEV, 43)
    pages = [torch.randint(0, 256, (L // S, H, S, D * w // 8), generator=g, dtype=torch.uint8) for w in widths]
    norms = [torch.rand(L // S, H, S, generator=g) * 0.5 + 2.0, torch.rand(L // S, H, S, generator=g) * 4 + 8.0]
    # the second token, of the same stream: the codes of the first's key, longer; scores of about 60 and 60 + lead (log2),
    # all others far below
    pages[0][second // S, :, second % S] = pages[0][first // S, :, first % S]
    norms[0][first // S, :, first % S] = 11.0
    norms[0][second // S, :, second % S] = 11.0 * (60 + lead) / 60
    pages, norms = [p.to(DEV) for p in pages], [n.half().to(DEV) for n in norms]
    kv = pa.PackedKV(pages[0], norms[0], pages[1], norms[1],
                     torch.arange(L // S, dtype=torch.int32, device=DEV).repeat(B, 1),
                     torch.full((B,), L, dtype=torch.int32, device=DEV), pa.Quantizer.from_tq(kq),
                     pa.Quantizer.from_tq(vq), D)
    scale = D ** -0.5
    k = plain.dequantised(pages[0], norms[0], kv.k_quant, kv.page_table[0], L, S, D)
    q = k[:, first] * (60 * math.log(2) / scale) / k[:, first].square().sum(-1, keepdim=True)
    q = q.repeat_interleave(4, 0)[None, :, None].expand(B, 4 * H, Q, D).half().contiguous()
    seen = torch.ones(Q, Q, dtype=torch.bool).tril().expand(B, Q, Q)
    got = tree_decode_attention(q, kv, plain.words(seen).to(DEV), scale).double()
    want = plain.tree_attention(q, kv, seen, scale)
    # How far each row's result is longer or shorter than it should be.  A probability is off by at most 2^-11 of itself;
    # with it in both sums the weights move by 2 w (1 - w) 2^-11, w <= 2^-lead the smaller weight.  Results are rounded
    # to fp16, which moves the length of 128 values by 2^-11 / sqrt(3) / sqrt(128) in the mean: four times that.
    w = 2.0 ** -lead
    bound = 2 * w * 2.0 ** -11 + 4 * 2.0 ** -11 / math.sqrt(3 * 128) + 1e-5
    longer = ((got * want).sum(-1) / want.square().sum(-1) - 1).abs()
    assert (longer <= bound).all(), f"{float(longer.max()):.2e} over {bound:.2e}"
