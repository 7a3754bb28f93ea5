"""What the operators of a drafted step refuse before anything is launched: at the C entry points with
addresses that nobody reads, and in Python on tensors without storage."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from winnow_b200 import _lib, packed_attention as pa
from winnow_b200.block_tables import DevicePages, TokenPlan, plan_tokens
from winnow_b200.packed_attention_cuda import tree_decode_attention
from winnow_b200.packed_backend import append_planned, keep_tokens
from winnow_b200.page_pool import PagePool
from winnow_b200.rotary import qk_norm_rope, rotary_table

ADDRESS = 1 << 20                              # never read: every call here ends at its checks


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield


def _tree(**kw):
    a = dict(q=ADDRESS, dtype=2, out=ADDRESS, table=ADDRESS, lens=ADDRESS, mask=ADDRESS, B=2, Hq=8, Hkv=2, Q=4, D=128,
             S=16, P=9, W=4, ws=ADDRESS, size=1 << 40, bw=4, pages=ADDRESS)
    a.update(kw)
    side = _lib.Side(a["pages"], ADDRESS, 1024, 1024, 16, 16, ADDRESS, None, ADDRESS, a["bw"])
    s3 = _lib.i64x(4096, 128, 1024)
    return _lib.lib().wtq_tree(a["q"], a["dtype"], s3, a["out"], s3, ctypes.byref(side), ctypes.byref(side), a["table"],
                               4, a["lens"], a["mask"], _lib.i64x(4, 1), 0.1, a["B"], a["Hq"], a["Hkv"], a["Q"], a["D"],
                               a["S"], a["P"], a["W"], a["ws"], a["size"], None, None)


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(mask=None),
                                 dict(dtype=3), dict(dtype=-1), dict(Hq=7), dict(Q=0), dict(D=0), dict(D=257), dict(S=0),
                                 dict(P=0), dict(W=0), dict(B=-1), dict(ws=None), dict(ws=ADDRESS + 64), dict(size=100),
                                 dict(bw=7), dict(bw=5, D=12), dict(pages=None), dict(B=1 << 20, Q=1 << 10),
                                 dict(B=1 << 13, Q=1 << 10, Hq=256, Hkv=2), dict(W=1 << 28, S=64)])
def test_tree_entry(bad):
    assert _tree(**bad) in (-1, -4)
    assert _lib.lib().wtq_last_error()


def test_tree_of_no_sequences_is_nothing():
    assert _tree(B=0) == 0


def test_where_the_tensor_cores_serve():
    def at(dtype=2, D=128, S=16, bk=4, bv=4, pages=ADDRESS, stride=1024, norm_stride=16):
        k, v = (_lib.Side(pages, ADDRESS, stride, 1024, norm_stride, 16, ADDRESS, None, ADDRESS, b) for b in (bk, bv))
        return _lib.lib().wtq_tree_on_tensor_cores(ctypes.byref(k), ctypes.byref(v), dtype, D, S)
    assert at() == at(dtype=1) == at(D=64) == at(bv=6) == at(bk=6, bv=6) == at(bk=8, bv=8) == at(S=64) == 1
    assert at(dtype=0) == at(D=96) == at(S=8) == at(S=24) == at(bk=6) == at(bk=3) == at(pages=ADDRESS + 8) == 0
    assert at(stride=1032) == at(norm_stride=4) == 0


def _rope(heads=(8, 2, 0), **kw):
    a = dict(x=ADDRESS, out=ADDRESS, dtype=2, wdtype=2, positions=ADDRESS, table=ADDRESS, rows=10, B=2, n=3, D=128, rot=128)
    a.update(kw)
    s = (_lib.RopeSide * 3)(*(_lib.RopeSide(a["x"], a["out"], _lib.i64x(1, 1, 1), _lib.i64x(1, 1, 1), None, h) for h in heads))
    return _lib.lib().wtq_qk_norm_rope(s, a["dtype"], a["wdtype"], 1e-6, a["positions"], 3, a["table"], 128, a["rows"],
                                       a["B"], a["n"], a["D"], a["rot"], 0, None, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(out=None), dict(dtype=9), dict(wdtype=-1), dict(positions=None),
                                 dict(table=None), dict(rows=-1), dict(B=-1), dict(n=-1), dict(D=0), dict(D=300),
                                 dict(rot=130), dict(rot=7), dict(rot=-2), dict(heads=(-1, 2, 0)), dict(B=1 << 20, n=1 << 20)])
def test_rope_entry(bad):
    assert _rope(**bad) == -1


def test_rope_of_nothing_is_nothing():
    assert _rope(B=0) == _rope(n=0) == _rope(heads=(0, 0, 0)) == 0


def _plan(**kw):
    a = dict(lengths=ADDRESS, new=ADDRESS, parents=None, table=ADDRESS, held=ADDRESS, free=ADDRESS, count=ADDRESS, B=3, W=4,
             S=16, tokens=9, drafted=0, stack=5, ticket=None, out=ADDRESS * 2, in_place=False, null=None)
    a.update(kw)
    names = [n for n, _ in _lib.Plan._fields_]
    out = {n: a["out"] + 4096 * i for i, n in enumerate(names)}
    if a["in_place"]:
        out["seq_lens"] = a["lengths"]
    if a["null"]:
        out[a["null"]] = None
    return _lib.lib().wtq_plan_tokens(a["lengths"], a["new"], a["parents"], 3, a["table"], 4, a["held"], a["free"], a["count"],
                                      a["B"], a["W"], a["S"], a["tokens"], a["drafted"], a["stack"],
                                      ctypes.byref(_lib.Plan(**out)), a["ticket"], None, None)


@pytest.mark.parametrize("bad", [dict(lengths=None), dict(new=None), dict(table=None), dict(held=None), dict(free=None),
                                 dict(count=None), dict(B=-1), dict(B=5000), dict(W=0), dict(S=0), dict(tokens=-1),
                                 dict(drafted=3), dict(parents=ADDRESS), dict(parents=ADDRESS, drafted=4), dict(stack=-1),
                                 dict(in_place=True), *(dict(null=n) for n, _ in _lib.Plan._fields_[:8]),
                                 dict(parents=ADDRESS, drafted=3, null="mask")])
def test_plan_entry(bad):
    assert _plan(**bad) == -1


def _keep(**kw):
    a = dict(pages=ADDRESS, norms=ADDRESS, row=64, table=ADDRESS, lens=ADDRESS, keep=ADDRESS, counts=ADDRESS, layers=1, B=2,
             Hkv=2, S=16, P=4, W=3, most=2, drafted=4, out=2 * ADDRESS)
    a.update(kw)
    side = _lib.PoolSide(a["pages"], a["norms"], 64, 64, 64, 16, 16, 16, a["row"])
    return _lib.lib().wtq_keep_tokens(ctypes.byref(side), ctypes.byref(side), a["table"], 3, a["lens"], a["keep"], 2,
                                      a["counts"], a["layers"], a["B"], a["Hkv"], a["S"], a["P"], a["W"], a["most"],
                                      a["drafted"], None, a["out"], None, None)


@pytest.mark.parametrize("bad", [dict(pages=None), dict(norms=None), dict(row=0), dict(table=None), dict(lens=None),
                                 dict(keep=None), dict(counts=None), dict(layers=0), dict(B=-1), dict(Hkv=0), dict(S=0),
                                 dict(P=0), dict(W=0), dict(most=-1), dict(drafted=-1), dict(out=None), dict(out=ADDRESS)])
def test_keep_entry(bad):
    assert _keep(**bad) == -1


def test_release_entry():
    r = _lib.lib().wtq_release_tokens
    assert r(None, ADDRESS, 4, ADDRESS, ADDRESS, ADDRESS, ADDRESS, 2, 4, 4, None, None) == -1
    assert r(ADDRESS, ADDRESS, 4, ADDRESS, ADDRESS, ADDRESS, ADDRESS, 9999, 4, 4, None, None) == -1
    assert r(None, None, 4, None, None, None, None, 0, 4, 4, None, None) == 0


# ---- Python ----------------------------------------------------------------------------------
def test_there_is_no_cpu_path():
    x = torch.zeros(1, 2, 3, 16)
    i = torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(_lib.BackendError):
        qk_norm_rope(x, x, i, rotary_table(16, 4, device="cpu"))
    j = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(_lib.BackendError):
        plan_tokens(j, j, i, j, i[0], j, 16, 2)
    with pytest.raises(_lib.BackendError):
        DevicePages(PagePool(num_layers=1, num_pages=4, num_kv_heads=1, page_size=16, nb_k=8, nb_v=8), "a", pages=1,
                    batch=1, width=1)
    pages, norms = torch.zeros(1, 4, 1, 16, 8, dtype=torch.uint8), torch.zeros(1, 4, 1, 16, dtype=torch.float16)
    with pytest.raises(_lib.BackendError):
        keep_tokens(pages, norms, pages, norms, i, j, i, j, 2)
    q = pa.Quantizer(torch.eye(16), torch.zeros(16), 4)
    kv = pa.PackedKV(pages[0], norms[0], pages[0], norms[0], i, j, q, q, 16)
    with pytest.raises(pa.UnsupportedLayout, match="CUDA"):
        tree_decode_attention(x, kv, torch.zeros(1, 3, 1, dtype=torch.int32), 1.0)


def _rope_call(**kw):
    e = lambda *s, dtype=torch.bfloat16, device="cuda": torch.empty(*s, dtype=dtype, device=device)     # noqa: E731
    a = dict(q=e(2, 8, 3, 64), k=e(2, 2, 3, 64), positions=e(2, 3, dtype=torch.int32), table=e(9, 64, dtype=torch.float32))
    a.update({k: v(e) for k, v in kw.items()})
    return qk_norm_rope(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("table"), **a)


@pytest.mark.parametrize("bad", [
    dict(k=lambda e: e(2, 2, 4, 64)), dict(k=lambda e: e(3, 2, 3, 64)), dict(k=lambda e: e(2, 2, 3, 64, dtype=torch.float16)),
    dict(q=lambda e: e(2, 8, 64)), dict(positions=lambda e: e(2, 3, dtype=torch.int64)),
    dict(positions=lambda e: e(2, 4, dtype=torch.int32)), dict(table=lambda e: e(9, 66, dtype=torch.float32)),
    dict(table=lambda e: e(9, 64)), dict(table=lambda e: e(9, 31, dtype=torch.float32)),
    dict(table=lambda e: e(64, 9, dtype=torch.float32).t()), dict(q_weight=lambda e: e(63)),
    dict(q_weight=lambda e: e(64), k_weight=lambda e: e(64, dtype=torch.float32)), dict(v=lambda e: e(2, 3, 3, 64)),
    dict(out=lambda e: (e(2, 8, 3, 64),)), dict(out=lambda e: (e(2, 8, 3, 64), e(2, 2, 3, 64, dtype=torch.float32)))])
def test_rope_arguments(fake, bad):
    with pytest.raises(ValueError):
        _rope_call(**bad)


@pytest.mark.parametrize("bad", [dict(q=lambda e: e(2, 8, 3, 64, dtype=torch.float64)), dict(k=lambda e: e(2, 2, 3, 64, device="cpu")),
                                 dict(table=lambda e: e(9, 64, dtype=torch.float32, device="cpu"))])
def test_rope_types_and_devices(fake, bad):
    with pytest.raises(_lib.BackendError):
        _rope_call(**bad)


def test_rope_has_no_backward_pass(fake):
    with pytest.raises(RuntimeError, match="backward"):
        _rope_call(q=lambda e: e(2, 8, 3, 64).requires_grad_())
    with pytest.raises(RuntimeError, match="backward"):
        _rope_call(q_weight=lambda e: e(64).requires_grad_())


def _plan_call(**kw):
    e = lambda *s, dtype=torch.int32, device="cuda": torch.empty(*s, dtype=dtype, device=device)        # noqa: E731
    a = dict(lengths=e(2), new_tokens=e(2), table=e(2, 4), held=e(2), free_pages=e(5), free_count=e(1), page_size=16, tokens=6)
    a.update({k: v(e) for k, v in kw.items()})
    return plan_tokens(**a)


@pytest.mark.parametrize("bad", [
    dict(lengths=lambda e: e(3)), dict(lengths=lambda e: e(2, dtype=torch.int64)), dict(new_tokens=lambda e: e(2, 1)),
    dict(new_tokens=lambda e: None), dict(parents=lambda e: e(2, 3)), dict(held=lambda e: e(4)[::2]),
    dict(table=lambda e: e(8)), dict(table=lambda e: e(4, 2).t()), dict(table=lambda e: e(1, 4).expand(2, 4)),
    dict(table=lambda e: e(2, 0)), dict(free_count=lambda e: e(2)), dict(free_pages=lambda e: e(5, dtype=torch.int64)),
    dict(page_size=lambda e: 0), dict(tokens=lambda e: -1), dict(new_tokens=lambda e: None, parents=lambda e: e(2, 4)),
    dict(new_tokens=lambda e: None, parents=lambda e: e(3, 3)), dict(new_tokens=lambda e: None, parents=lambda e: e(3, 2).t()),
    dict(out=lambda e: TokenPlan(e(2), e(2), e(1), e(3), e(6), e(6), e(6), e(6), None)),
    dict(out=lambda e: TokenPlan(e(2), e(2), e(1), e(2), e(6), e(6), e(6, 1), e(6), None))])
def test_plan_arguments(fake, bad):
    with pytest.raises(ValueError):
        _plan_call(**bad)


def test_plan_devices(fake):
    for bad in (dict(held=lambda e: e(2, device="cpu")), dict(status=lambda e: e(1, device="cpu")),
                dict(ticket=lambda e: e(1, device="cpu"))):
        with pytest.raises(_lib.BackendError):
            _plan_call(**bad)


def test_planned_append_needs_the_plans_tokens(fake):
    e = torch.empty
    p = TokenPlan(*[None] * 6, e(6, 1, dtype=torch.int32), e(6, dtype=torch.int32), None)
    for shape in ((5, 2, 64), (6, 2, 1, 64)):
        with pytest.raises(ValueError):
            append_planned(e(*shape), e(*shape), None, None, None, None, p, None, None)
