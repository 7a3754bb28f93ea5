"""How far 16-bit results of drafted trees' attention are from 64 bits, beyond the rounding of the result itself.

A value rounded to nearest in fp16 is off by at most 2^-11 of itself, in the mean of many by 2^-11 / sqrt(3) = 2.82e-4 or
less.  That happens to a probability once; with bf16 results also to a value twice (the centroid, its product with the
norm) and to a joined state.  Scores are products of split operands, off by 2^-21 of |q| |k| at most, which is below 1e-4 nats for the largest
logits here (100 nats).  So beside its own rounding, measured on the exact result, an fp16 result is off by
2.82e-4 + 0.2e-4 and a bf16 result by sqrt(4) 2.82e-4 + 0.2e-4 of its norm; 1 % is left for the spread of
a mean over some 10^5 elements.
"""
import pytest
import torch

import plain
from test_gpu_tree import DEV, build, trees
from winnow_b200.packed_attention_cuda import tree_decode_attention

pytestmark = pytest.mark.gpu
BESIDE = {torch.float16: 3.0e-4, torch.bfloat16: 5.9e-4}


@pytest.mark.parametrize("mult", [0.5, 1.0, 2.0, 3.0, 4.0, 5.0])
@pytest.mark.parametrize("D,widths", [(128, (4, 4)), (128, (4, 6)), (128, (8, 8)), (64, (6, 6)), (64, (4, 4))])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_error_beside_the_results_rounding(dtype, D, widths, mult):
    """Logits of half a nat to several nats, where tiles' best scores lie anywhere up to some tens."""
    lens, Hq, Q = [3000, 500, 9000], 16, 16
    kv = build(lens, 2, D, 16, *widths)
    g = torch.Generator().manual_seed(7)
    q = (mult * torch.randn(3, Q, Hq, D, generator=g)).to(DEV, dtype).transpose(1, 2)
    seen = trees(3, Q, 4)
    got = tree_decode_attention(q, kv, plain.words(seen).to(DEV), D ** -0.5)
    want = plain.tree_attention(q, kv, seen, D ** -0.5)
    own = (want.to(dtype).double() - want).norm() / want.norm()
    err = (got.double() - want).norm() / want.norm()
    assert err <= 1.01 * (own ** 2 + BESIDE[dtype] ** 2) ** 0.5, f"{err:.3e}, own rounding {own:.3e}"
