"""Pages of a batch on the device after they have been given back: nothing may use them, another request may hold them."""
import pytest
import torch

from winnow_b200.block_tables import DevicePages
from winnow_b200.cache import _get_quantizer
from winnow_b200.engine_step import TreeSession
from winnow_b200.page_pool import PagePool, StalePage

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pool_and_pages():
    pool = PagePool(num_layers=2, num_pages=8, num_kv_heads=1, page_size=16, nb_k=32, nb_v=32, device=torch.device(DEV))
    return pool, DevicePages(pool, "batch", pages=8, batch=2, width=4)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("how", ["close", "release"])
def test_nothing_uses_pages_that_were_given_back(how):
    pool, pages = pool_and_pages()
    quant = _get_quantizer(4, 64, DEV, 42)
    session = TreeSession(pages, k_quant=quant, v_quant=quant, head_dim=64, q_heads=2, dtype=torch.bfloat16, drafted=2)
    pages.extend(i32([20, 3]), tokens=23)
    session.begin(i32([[-1, 0], [-1, -2]]))
    assert (pages.close() if how == "close" else pool.release("batch")) == 8
    torch.cuda.synchronize()
    pool.ensure("other", 8 * 16)
    before = [t.clone() for t in (pool.k_pages, pool.k_norms, pool.v_pages, pool.v_norms)]
    x = torch.randn(2, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: pages.extend(i32([1, 1]), tokens=2), lambda: pages.extend(parents=i32([[-1], [-1]])),
                 lambda: pages.keep(i32([[0], [0]]), i32([1, 0]), 2), lambda: pages.release(i32([1, 0])),
                 lambda: session.begin(i32([[-1, 0], [-1, 0]])), lambda: session.layer(0, x, x, x.expand(2, 2, 2, 64)),
                 lambda: session.accept(i32([[0], [0]]), i32([1, 0]))):
        with pytest.raises(StalePage):
            call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (pool.k_pages, pool.k_norms, pool.v_pages, pool.v_norms)))


def test_closing_twice_leaves_the_next_batch_alone():
    pool, pages = pool_and_pages()
    assert pages.close() == 8
    torch.cuda.synchronize()
    again = DevicePages(pool, "batch", pages=8, batch=2, width=4)
    assert pages.close() == 0
    again.extend(i32([20, 3]), tokens=23)
    again.check()
    assert again.close() == 8
