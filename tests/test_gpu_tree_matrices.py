"""Drafted trees' attention with matrices that are no rotations: any scale, elements above fp16's range times 2^-8."""
import pytest
import torch

from test_gpu_tree import DEV, build, check
from winnow_b200 import packed_attention as pa

pytestmark = pytest.mark.gpu


def scaled(kv, factor, k_norms):
    """Both sides' matrices times `factor`, with keys' norms scaled so that the logits keep their size."""
    quants = [pa.Quantizer(q.Pi.contiguous() * factor, q.centroids, q.bit_width) for q in (kv.k_quant, kv.v_quant)]
    return pa.PackedKV(kv.k_pages, (kv.k_norms.float() * k_norms).half(), kv.v_pages, kv.v_norms, kv.page_table, kv.seq_lens,
                       *quants, kv.head_dim)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("factor", [2.0 ** 11, 2.0 ** -4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matrices_of_any_scale(dtype, factor, D):
    """Norms times powers of two are as exact as before, and so are the bounds."""
    kv = scaled(build([400, 130], 2, D, 16, 4, 4), factor, 1 / factor)
    check(kv, 2, 8, 6, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_matrices_that_are_small(dtype):
    """Elements of 1e-7, queries that make up for it: parts below fp16's smallest numbers if they were not scaled up."""
    kv = scaled(build([400, 130], 2, 128, 16, 4, 4), 2.0 ** -20, 1.0)
    check(kv, 2, 8, 6, dtype, mult=2.0 ** 20)


def test_a_few_large_elements():
    kv = scaled(build([400, 130], 2, 128, 16, 4, 4), 1.0, 1.0)
    for quant in (kv.k_quant, kv.v_quant):
        quant.Pi[3, 5] = 1000.0
    check(kv, 2, 8, 6, torch.float32, mult=1e-3)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Hq,Q", [(1, 1, 1), (1, 3, 5), (2, 6, 21), (3, 14, 19)])
def test_rows_that_leave_part_of_a_block_empty(B, Hq, Q, D):
    """Blocks of 16 to 128 rows: lanes past the last one load with the others and store nothing."""
    kv = build([90] * B, 1, D, 16, 4, 4)
    for dtype in (torch.float32, torch.float16):
        check(kv, B, Hq, Q, dtype)
