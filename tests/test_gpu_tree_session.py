"""A run of the step's operators together, as a server uses them: plan, norms with rotation, append, tree
attention, accepted path, over many steps, against the definitions and against plain decoding."""
import random

import pytest
import torch

import plain
from winnow_b200 import _lib, packed_attention as pa
from winnow_b200.block_tables import DevicePages
from winnow_b200.cache import _get_quantizer
from winnow_b200.engine_step import DecodeSession, TreeSession
from winnow_b200.packed_backend import append_planned
from winnow_b200.page_pool import PagePool, PoolExhausted, StalePage
from winnow_b200.rotary import Rotary, qk_norm_rope, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda"
B, HQ, HKV, D, S, LAYERS = 3, 8, 4, 128, 16, 2


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def build(dtype, pages=60, drafted=9):
    kq, vq = _get_quantizer(4, D, DEV, 42), _get_quantizer(4, D, DEV, 43)
    pool = PagePool(num_layers=LAYERS, num_pages=pages + 4, num_kv_heads=HKV, page_size=S, nb_k=64, nb_v=64, device=DEV)
    g = torch.Generator().manual_seed(1)
    weights = [[(1 + 0.2 * torch.randn(D, generator=g)).to(DEV, dtype) for _ in range(LAYERS)] for _ in range(2)]
    rotary = Rotary(rotary_table(D, 400, base=1e6), *weights)
    d = DevicePages(pool, "batch", pages=pages, batch=B, width=20)
    return pool, d, TreeSession(d, k_quant=kq, v_quant=vq, head_dim=D, q_heads=HQ, dtype=dtype, drafted=drafted,
                                rotary=rotary), rotary, kq, vq


def projections(tokens, layer, dtype):
    """What a projection gives for tokens with these ids: the same for the same id."""
    out = torch.empty(len(tokens), len(tokens[0]), HQ + 2 * HKV, D)
    for b, row in enumerate(tokens):
        for i, t in enumerate(row):
            out[b, i] = torch.randn(HQ + 2 * HKV, D, generator=torch.Generator().manual_seed(1000 * t + layer))
    out = out.to(DEV, dtype).transpose(1, 2)
    return out[:, :HQ], out[:, HQ:HQ + HKV], out[:, HQ + HKV:]


def prompt(d, kq, vq, rotary, tokens, dtype):
    """Ragged prompts in one step: rotate and append what each sequence has."""
    new = [len(t) for t in tokens]
    p = d.extend(i32(new), tokens=sum(new))
    flat = [[t] for row in tokens for t in row]
    for layer in range(LAYERS):
        q, k, v = projections(flat, layer, dtype)
        _, k = rotary.apply(layer, q, k, p.positions.view(-1, 1))
        append_planned(k[:, :, 0], v[:, :, 0], *d.pool.layer(layer), p, kq, vq, status=d.status)
    d.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_speculative_steps_leave_what_plain_decoding_leaves(dtype):
    rng = random.Random(3)
    pool, d, s, rotary, kq, vq = build(dtype)
    texts = [[rng.randrange(10 ** 6) for _ in range(n)] for n in (5, 33, 16)]
    prompt(d, kq, vq, rotary, texts, dtype)
    for step in range(5):
        parents, drafts = [], []
        for b in range(B):
            real = 9 - rng.choice((0, 0, 3))
            parents.append([-1 if i == 0 else rng.randrange(max(0, i - 4), i) if i < real else -2 for i in range(9)])
            drafts.append([rng.randrange(10 ** 6) for _ in range(9)])
        before = d.lengths.tolist()
        assert before == [len(t) for t in texts]
        p = s.begin(i32(parents))
        seen = plain.reach(parents)
        depth = seen.sum(-1) - 1
        want = torch.where(depth >= 0, torch.tensor(before)[:, None] + depth, -1)
        assert torch.equal(p.positions.view(B, 9).cpu().long(), want)
        for layer in range(LAYERS):
            q, k, v = projections(drafts, layer, dtype)
            out = s.layer(layer, k, v, q)
            ref_q = plain.norm_rope(q, p.positions.view(B, 9), rotary.table, rotary.q_weights[layer], 1e-6, False)
            assert (s.q_in.double() - ref_q).norm() <= torch.finfo(dtype).eps * ref_q.norm()
            kv = pa.PackedKV(*pool.layer(layer), d.table, d.lengths, pa.Quantizer.from_tq(kq), pa.Quantizer.from_tq(vq), D)
            exact = plain.tree_attention(s.q_in, kv, seen, D ** -0.5)
            assert (out.double() - exact).norm() <= (2e-5 if dtype == torch.float32 else 4e-3) * exact.norm()
            # the drafted tokens' codes are those of the staged keys, at the places the plan says
            codes, norms = kq.quantize(s.k_in.float().permute(0, 2, 1, 3).reshape(-1, D).contiguous(), packed=True,
                                       order=_lib.ORDER_SEQUENTIAL)
            at = (p.slot_pages[:, 0].long(), p.slot_ends.long() - 1)
            assert torch.equal(pool.k_pages[layer][at[0], :, at[1]], codes.view(B * 9, HKV, -1))
            assert torch.equal(pool.k_norms[layer][at[0], :, at[1]], norms.half().view(B * 9, HKV))
        # accept a path from the root down
        paths = []
        for b in range(B):
            leaf = rng.choice([i for i in range(9) if parents[b][i] >= -1])
            paths.append(seen[b, leaf].nonzero().flatten().tolist())
            texts[b] += [drafts[b][i] for i in paths[b]]
        lengths = s.accept(i32([x + [-1] * (9 - len(x)) for x in paths]), i32([len(x) for x in paths]))
        assert lengths.tolist() == [len(t) for t in texts]
        d.check()
    # the same texts, token by token
    pool2 = PagePool(num_layers=LAYERS, num_pages=60, num_kv_heads=HKV, page_size=S, nb_k=64, nb_v=64, device=DEV)
    owners = [f"r{b}" for b in range(B)]
    plain_session = DecodeSession(pool2, owners, [0] * B, k_quant=kq, v_quant=vq, head_dim=D, q_heads=HQ, dtype=dtype,
                                  max_tokens=200, rotary=rotary)
    for i in range(min(len(t) for t in texts)):
        plain_session.begin_step()
        for layer in range(LAYERS):
            q, k, v = projections([[t[i]] for t in texts], layer, dtype)
            plain_session.layer(layer, k, v, q)
    plain_session.check()
    n = min(len(t) for t in texts)
    for b in range(B):
        for layer in range(LAYERS):
            for x, y in zip(pool.layer(layer), pool2.layer(layer)):
                rows = [z[t[b, :-(-n // S)].long()].transpose(0, 1).flatten(1, 2)[:, :n]
                        for z, t in ((x, d.table), (y, plain_session.table.table))]
                assert torch.equal(*rows)
    assert d.close() == 60


def test_a_captured_step_is_replayed():
    dtype = torch.bfloat16
    pool, d, s, rotary, kq, vq = build(dtype)
    prompt(d, kq, vq, rotary, [[1, 2, 3], [4] * 20, [5, 6]], dtype)
    parents = i32([[-1, 0, 0, 1, 1, 2, 3, 4, 5]] * B)
    keep, counts = i32([[0, 2, 5]] * B), i32([3, 0, 2])
    inputs = [[t.contiguous() for t in projections([[7 + i for i in range(9)]] * B, layer, dtype)] for layer in range(LAYERS)]

    def step():
        s.begin(parents)
        outs = [s.layer(layer, k, v, q).clone() for layer, (q, k, v) in enumerate(inputs)]
        s.accept(keep, counts)
        return outs

    step()                                                   # everything that is made once exists now
    start = [t.clone() for t in (d.lengths, d.held, d.free_count, d.table, *pool.layer(0), *pool.layer(1))]

    def restore():
        for t, x in zip((d.lengths, d.held, d.free_count, d.table, *pool.layer(0), *pool.layer(1)), start):
            t.copy_(x)

    want = step()
    after = [t.clone() for t in (d.lengths, d.held, d.free_count, *pool.layer(0), *pool.layer(1))]
    restore()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    restore()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip((d.lengths, d.held, d.free_count, *pool.layer(0), *pool.layer(1)), after))
    d.check()


def test_slots_without_a_request_and_an_exhausted_pool():
    pool, d, s, rotary, kq, vq = build(torch.bfloat16, pages=4)
    parents = i32([[-1] + [0] * 8, [-2] * 9, [-2] * 9])
    for _ in range(3):
        p = s.begin(parents)
        q, k, v = projections([[1] * 9] * B, 0, torch.bfloat16)
        out = s.layer(0, k, v, q)
        assert not out[1:].any() and out[0].any()
        s.accept(i32([[0, 1]] * B), i32([2, 0, 0]))
    assert d.lengths.tolist() == [6, 0, 0] and (p.positions.view(B, 9)[1:] == -1).all()
    d.check()
    d.extend(i32([0, 0, 60]), tokens=60)
    with pytest.raises(PoolExhausted):
        d.check()
    assert d.lengths.tolist() == [6, 0, 0]
    with pytest.raises(ValueError):
        s.begin(i32([[-1]] * B))
    with pytest.raises(RuntimeError):
        s.layer(0, k, v, q)
    with pytest.raises(ValueError):
        DevicePages(pool, "batch", pages=1, batch=1, width=1)
    with pytest.raises(PoolExhausted):
        DevicePages(pool, "other", pages=10, batch=1, width=1)


def test_decode_session_with_rotary_and_a_graph():
    """Rotation in the staging launch: the same outputs as rotating first, with and without graphs."""
    kq, vq = _get_quantizer(4, D, DEV, 42), _get_quantizer(4, D, DEV, 43)
    rotary = Rotary(rotary_table(D, 100))
    outs = []
    for mode in range(3):
        pool = PagePool(num_layers=LAYERS, num_pages=12, num_kv_heads=HKV, page_size=S, nb_k=64, nb_v=64, device=DEV)
        s = DecodeSession(pool, ["a", "b"], [0, 0], k_quant=kq, v_quant=vq, head_dim=D, q_heads=HQ,
                          dtype=torch.bfloat16, max_tokens=64, rotary=None if mode == 0 else rotary)
        got = []
        for i in range(4):
            s.begin_step()
            if mode == 2 and i == 1:
                s.capture()
            for layer in range(LAYERS):
                q, k, v = projections([[i], [100 + i]], layer, torch.bfloat16)
                if mode == 0:
                    q, k = qk_norm_rope(q, k, torch.full((2, 1), i, dtype=torch.int32, device=DEV), rotary.table)
                got.append(s.layer(layer, k, v, q).clone())
        s.check()
        outs.append(torch.stack(got))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_a_position_past_the_table_is_reported():
    pool, d, s, rotary, kq, vq = build(torch.bfloat16)
    s.rotary = Rotary(rotary_table(D, 2))
    s.begin(i32([[-1, 0, 1, 2, 3, 4, 5, 6, 7]] * B))
    q, k, v = projections([[1] * 9] * B, 0, torch.bfloat16)
    s.layer(0, k, v, q)
    with pytest.raises(StalePage):
        s.check()


def test_a_refused_step_leaves_the_histories():
    """More pages than are free: nothing is appended, kept or cut off, and the step says so."""
    pool, d, s, rotary, kq, vq = build(torch.bfloat16, pages=6)
    prompt(d, kq, vq, rotary, [[1] * 30, [2] * 31, [3] * 29], torch.bfloat16)
    def state():
        return [t.clone() for t in (d.lengths, d.held, d.free_count, d.table, *pool.layer(0), *pool.layer(1))]
    before = state()
    p = s.begin(i32([[-1, 0, 1, 2, 3, 4, 5, 6, 7]] * B))
    q, k, v = projections([[1] * 9] * B, 0, torch.bfloat16)
    for layer in range(LAYERS):
        assert not s.layer(layer, k, v, q).any()
    assert s.accept(i32([[0, 1]] * B), i32([2, 1, 0])).tolist() == [30, 31, 29]
    assert all(torch.equal(a, b) for a, b in zip(state(), before)) and not p.mask.any()
    with pytest.raises(PoolExhausted):
        s.check()
    with pytest.raises(RuntimeError):
        s.accept(i32([[0, 1]] * B), i32([2, 1, 0]))


def test_a_step_without_a_rotary_takes_any_strides():
    _, d, s, _, kq, vq = build(torch.float32)
    s.rotary = None
    parents = i32([[-1, 0, 1, 1, 3, 0, 5, 6, -2]] * B)
    outs = []
    q, k, v = projections([[i + 10 * b for i in range(9)] for b in range(B)], 0, torch.float32)
    for make in (lambda t: t, lambda t: t.contiguous()):
        s.begin(parents)
        outs.append(s.layer(0, make(k), make(v), make(q)).clone())
        s.accept(i32([[0]] * B), i32([0] * B))
    s.check()
    assert torch.equal(*outs) and outs[0].any()


def test_padding_that_is_not_a_number_reaches_nobody():
    """The projections of padding hold whatever they hold."""
    pool, d, s, rotary, kq, vq = build(torch.bfloat16)
    parents = i32([[-1, 0, 1, 1, 3, 0, 5, -2, -2], [-2] * 9, [-1, 0, -2, 0, -2, -2, 0, 6, -2]])
    outs = []
    for bad in (0.0, float("nan"), float("inf")):
        p = s.begin(parents)
        q, k, v = projections([[i + 10 * b for i in range(9)] for b in range(B)], 0, torch.bfloat16)
        for t in (q, k, v):
            t.transpose(1, 2)[parents == -2] = bad
        outs.append(s.layer(0, k, v, q).clone())
        s.accept(i32([[0]] * B), i32([0] * B))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and outs[0].isfinite().all()
