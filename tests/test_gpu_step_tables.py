"""Block tables, slot maps, masks and kept paths of a drafted step: whole numbers and moved bytes, all equal."""
import random

import pytest
import torch

import plain
from winnow_b200 import _lib
from winnow_b200.block_tables import DevicePages, TokenPlan, plan_tokens
from winnow_b200.packed_backend import keep_tokens
from winnow_b200.page_pool import PagePool, PoolExhausted

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def setting(B, S, rng, longest, spare, width=None):
    lens = [rng.choice((0, 1, S - 1, S, S + 1, rng.randint(0, longest))) for _ in range(B)]
    lens = [min(n, longest) for n in lens]
    held = [-(-n // S) + (rng.random() < 0.2) for n in lens]
    W = width or max(held) + 70
    ids = list(range(sum(held) + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (W - h))
        at += h
    return lens, held, table, ids[at:]


def compare(p, want, table, want_table):
    for name, value in want.items():
        assert getattr(p, name).flatten().tolist() == value, name
    assert table.tolist() == want_table


@pytest.mark.parametrize("B,S,longest,most", [(1, 16, 40, 1), (3, 1, 5, 4), (7, 16, 100, 40), (64, 32, 500, 3),
                                              (300, 7, 60, 20), (1025, 16, 90, 2), (5, 64, 9000, 3000)])
@pytest.mark.parametrize("room", [0, 5])
def test_ragged_steps(B, S, longest, most, room):
    rng = random.Random(B * 100 + room)
    lens, held, table, free = setting(B, S, rng, longest, spare=B * (most // S + 2), width=(longest + most) // S + 3)
    new = [rng.randint(0, most) for _ in range(B)]
    tokens = sum(new) + room
    t = i32(table)
    p = plan_tokens(i32(lens), i32(new), t, i32(held), i32(free), i32([len(free)]), S, tokens)
    want = plain.plan(lens, new, table, held, free, len(free), S, tokens)
    compare(p, want, t, table)
    assert p.mask is None


@pytest.mark.parametrize("B,Q", [(1, 1), (2, 31), (5, 32), (9, 33), (3, 100), (257, 7)])
def test_trees(B, Q):
    rng = random.Random(Q)
    lens, held, table, free = setting(B, 16, rng, 200, spare=B * (Q // 16 + 2))
    parents = [[-1 if i == 0 or rng.random() < 0.1 else -2 if rng.random() < 0.1 else rng.randint(max(0, i - 9), i - 1)
                for i in range(Q)] for _ in range(B)]
    t, status = i32(table), i32([0])
    p = plan_tokens(i32(lens), None, t, i32(held), i32(free), i32([len(free)]), 16, B * Q, parents=i32(parents),
                    status=status)
    compare(p, plain.plan(lens, None, table, held, free, len(free), 16, B * Q, parents), t, table)
    assert torch.equal(p.mask.cpu(), plain.words(plain.reach(parents)))
    assert int(status) == 0


def test_parents_behind_their_children_are_padding():
    parents = [[-1, 0, 2, 7, -5, 1]]
    status = i32([0])
    p = plan_tokens(i32([3]), None, i32([[0] + [-1] * 3]), i32([1]), i32([1, 2]), i32([2]), 16, 6, parents=i32(parents),
                    status=status)
    assert int(status) == _lib.STATUS_BAD_PARENT
    assert torch.equal(p.mask.cpu(), plain.words(plain.reach(parents)))
    assert p.positions.tolist() == [3, 4, -1, -1, -1, 5]


def refused(p, lens, held, count, status, bit):
    assert int(status) == bit
    assert p.seq_lens.tolist() == lens and p.held.tolist() == held and p.free_count.tolist() == [count]
    assert set(p.starts.tolist()) == {0}
    for t in (p.sequence, p.positions, p.slot_pages):
        assert (t == -1).all()
    assert not p.slot_ends.any()


@pytest.mark.parametrize("why", ["pages", "width", "tokens", "negative", "held", "count", "far"])
def test_refused_steps_take_nothing(why):
    lens, held, new, count, tokens, W = [20, 5], [2, 1], [30, 3], 4, 40, 8
    S, bit = 16, _lib.STATUS_BAD_POSITION
    if why == "pages":
        count, bit = 1, _lib.STATUS_NO_PAGES
    elif why == "width":
        W, bit = 3, _lib.STATUS_NO_PAGES
    elif why == "tokens":
        tokens = 32
    elif why == "negative":
        lens = [20, -1]
    elif why == "held":
        held = [2, 9]
    elif why == "far":
        lens, S, W = [2 ** 31 - 20, 5], 2 ** 28, 8
    else:
        count = 5
    free = [9, 8, 7, 6]
    t, status = torch.full((2, W), -1, dtype=torch.int32, device=DEV), i32([0])
    p = plan_tokens(i32(lens), i32(new), t, i32(held), i32(free), i32([count]), S, tokens, status=status)
    refused(p, lens, held, count, status, bit)
    assert (t == -1).all()


def test_refused_trees_see_nothing():
    status = i32([0])
    t = torch.full((2, 8), -1, dtype=torch.int32, device=DEV)
    p = plan_tokens(i32([16, 16]), None, t, i32([1, 1]), i32([3]), i32([1]), 16, 8, parents=i32([[-1, 0, 0, 1]] * 2),
                    status=status)
    refused(p, [16, 16], [1, 1], 1, status, _lib.STATUS_NO_PAGES)
    assert not p.mask.any()


def test_strided_tables_and_parents():
    t = torch.full((3, 9), -5, dtype=torch.int32, device=DEV)
    view = t[:, 2:7]
    parents = torch.full((3, 6), -9, dtype=torch.int32, device=DEV)
    parents[:, 1:5] = i32([-1, 0, 0, 2])
    p = plan_tokens(i32([15, 0, 32]), None, view, i32([1, 0, 2]), i32([4, 5, 6, 7]), i32([4]), 16, 12,
                    parents=parents[:, 1:5])
    assert p.held.tolist() == [2, 1, 3] and view[:, 0].tolist() == [-5, 6, -5] and view[:, 1].tolist() == [7, -5, -5]
    assert int(view[2, 2]) == 5 and (t[:, :2] == -5).all() and (t[:, 7:] == -5).all()


def pool_of(pages, layers=2, S=16, dev=DEV):
    return PagePool(num_layers=layers, num_pages=pages, num_kv_heads=2, page_size=S, nb_k=64, nb_v=96, device=dev)


def test_device_pages_over_many_steps():
    """Sequences come, grow by ragged and drafted steps, and go; a host model of the stack agrees throughout."""
    rng = random.Random(4)
    pool = pool_of(60)
    pool.ensure("somebody else", 5 * 16)
    B, S = 6, 16
    d = DevicePages(pool, "batch", pages=40, batch=B, width=12)
    ids = [ref.page for ref in pool.held("batch")]
    free, count = ids[::-1], 40
    lens, held, table = [0] * B, [0] * B, [[-1] * 12 for _ in range(B)]
    for step in range(30):
        if step % 3 == 2:
            parents = [[-1] + [rng.randint(0, i) for i in range(6)] for _ in range(B)]
            want = plain.plan(lens, None, table, held, free, count, S, 7 * B, parents)
            p = d.extend(parents=i32(parents))
            if want is not None:
                assert torch.equal(p.mask.cpu(), plain.words(plain.reach(parents)))
        else:
            new = [rng.randint(0, 9) for _ in range(B)]
            want = plain.plan(lens, new, table, held, free, count, S, sum(new))
            p = d.extend(i32(new), tokens=sum(new))
        if want is None:
            with pytest.raises(PoolExhausted):
                d.check()
        else:
            compare(p, want, d.table, table)
            lens, held, count = want["seq_lens"], want["held"], want["free_count"][0]
            d.check()
        if step % 7 == 6:
            marks = [int(rng.random() < 0.4) for _ in range(B)]
            d.release(i32(marks))
            for b in range(B):
                if marks[b]:
                    for c in reversed(range(held[b])):
                        free[count] = table[b][c]
                        table[b][c] = -1
                        count += 1
                    lens[b] = held[b] = 0
            assert d.free_pages[:count].tolist() == free[:count]
        assert d.lengths.tolist() == lens and d.held.tolist() == held and d.free_count.tolist() == [count]
        assert sorted(free[:count] + [x for row in table for x in row if x >= 0]) == sorted(ids)
    assert d.close() == 40 and pool.stats()["requests"] == 1


def test_in_place_over_many_blocks():
    """A step of many blocks that advances its own inputs, thirty times over."""
    B = 200
    lens, held, table = [0] * B, [0] * B, [[-1] * 80 for _ in range(B)]
    free = list(range(16000))
    rng = random.Random(1)
    t, L, h, c, ticket = i32(table), i32(lens), i32(held), i32([16000]), i32([0])
    fr = i32(free)
    count = 16000
    for _ in range(30):
        new = [rng.randint(0, 40) for _ in range(B)]
        n = sum(new)
        e = lambda *s: torch.empty(s, dtype=torch.int32, device=DEV)                     # noqa: E731
        out = TokenPlan(L, h, c, e(B + 1), e(n), e(n), e(n, 1), e(n), None)
        p = plan_tokens(L, i32(new), t, h, fr, c, 16, n, out=out, ticket=ticket)
        want = plain.plan(lens, new, table, held, free, count, 16, n)
        compare(p, want, t, table)
        assert int(ticket) == 0
        lens, held, count = want["seq_lens"], want["held"], want["free_count"][0]


def test_rooms_of_ragged_steps():
    """Any number of tokens, and no more tensors kept than there are powers of two."""
    d = DevicePages(pool_of(200), "batch", pages=200, batch=2, width=100)
    for n in [*range(0, 40), 100, 64, 65]:
        p = d.extend(i32([n - n // 3, n // 3]), tokens=n)
        assert p.slot_pages.shape == (n, 1) and p.sequence.tolist() == [0] * (n - n // 3) + [1] * (n // 3)
    assert len(d._room) <= 8
    d.check()


def test_captured_steps():
    pool = pool_of(200)
    d = DevicePages(pool, "batch", pages=200, batch=3, width=60)
    new = i32([0, 0, 0])
    d.extend(new, tokens=12)                                # the plan's tensors exist before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = d.extend(new, tokens=12)
    lens = [0, 0, 0]
    for step in ([5, 0, 7], [4, 4, 4], [0, 0, 0], [1, 2, 3]):
        new.copy_(i32(step))
        graph.replay()
        lens = [a + b for a, b in zip(lens, step)]
        assert d.lengths.tolist() == lens
        assert p.sequence.tolist() == [b for b in range(3) for _ in range(step[b])] + [-1] * (12 - sum(step))
    d.check()


# ---- kept paths --------------------------------------------------------------------------------
def random_pool(P, layers, Hkv, S, nb_k, nb_v, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda nb: torch.randint(0, 256, (layers, P, Hkv, S, nb), generator=g, dtype=torch.uint8).to(DEV)  # noqa: E731
    n = lambda: torch.randn(layers, P, Hkv, S, generator=g).half().to(DEV)                                  # noqa: E731
    return [r(nb_k), n(), r(nb_v), n()]


@pytest.mark.parametrize("B,drafted,S,layers,Hkv,nb", [(1, 1, 16, 1, 1, (64, 64)), (3, 8, 16, 2, 2, (64, 96)),
                                                       (4, 40, 16, 1, 3, (32, 48)), (2, 100, 64, 2, 1, (128, 64)),
                                                       (5, 9, 3, 2, 2, (10, 7)), (2, 70, 32, 1, 2, (20, 36))])
def test_kept_paths(B, drafted, S, layers, Hkv, nb):
    rng = random.Random(drafted)
    lens = [drafted + rng.randint(0, 50) for _ in range(B)]
    need = [-(-L // S) for L in lens]
    ids = list(range(sum(need) + 2))
    rng.shuffle(ids)
    W = max(need)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (W - n))
        at += n
    pool = random_pool(len(ids), layers, Hkv, S, *nb, seed=drafted)
    for trial in range(4):
        counts = [rng.randint(0, drafted) if trial else drafted for _ in range(B)]
        if trial == 1:
            counts[0] = 0
        paths = [sorted(rng.sample(range(drafted), c)) + [-1] * (drafted - c) for c in counts]
        want, lengths = plain.keep(pool, table, lens, paths, counts, drafted, S)
        status = i32([0])
        got = keep_tokens(*pool, i32(table), i32(lens), i32(paths), i32(counts), drafted, status=status)
        assert got.tolist() == lengths and int(status) == 0
        for a, b in zip(pool, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("path,count,lens", [([1, 1], 2, 20), ([2, 1], 2, 20), ([0, 8], 2, 20), ([-1, 0], 2, 20),
                                             ([0, 1], 3, 20), ([0, 1], -1, 20), ([0, 1], 2, 5), ([0, 1], 2, 99)])
def test_malformed_paths_move_nothing(path, count, lens):
    pool = random_pool(4, 2, 2, 16, 64, 64, 1)
    before = [t.clone() for t in pool]
    status = i32([0])
    got = keep_tokens(*pool, i32([[0, 1], [2, 3]]), i32([lens, 30]), i32([path, [0, 3]]), i32([count, 1]), 8,
                      status=status)
    assert got.tolist() == [lens - 8 if lens >= 8 else lens, 23]
    assert int(status) == _lib.STATUS_BAD_POSITION
    assert all(torch.equal(a, b) for a, b in zip(pool, before))


def test_pages_outside_the_pool_are_left_alone():
    pool = random_pool(3, 1, 2, 16, 64, 64, 1)
    before = [t.clone() for t in pool]
    status = i32([0])
    table = i32([[0, 5], [1, 2]])
    got = keep_tokens(*pool, table, i32([24, 24]), i32([[0, 7], [0, 7]]), i32([2, 2]), 12, status=status)
    assert got.tolist() == [14, 14] and int(status) == _lib.STATUS_BAD_PAGE
    want, _ = plain.keep(before, table.tolist(), [24, 24], [[0, 0], [0, 7]], [1, 2], 12, 16)
    assert all(torch.equal(a, b) for a, b in zip(pool, want))


def test_keep_strided_pools():
    """Layers, pages and heads inside wider buffers, rows off 16-byte borders."""
    S, D = 16, 64
    wide = torch.randint(0, 256, (2, 5, 3, S * D + 4), dtype=torch.uint8, device=DEV)
    pages = wide[:, :, :2, 4:].unflatten(3, (S, D))
    norms = torch.randn(2, 5, 3, S, device=DEV).half()[:, :, :2]
    rest = random_pool(5, 2, 2, S, 64, 64, 2)
    pool = [pages, norms, rest[2], rest[3]]
    before = wide.clone()
    want, lengths = plain.keep(pool, [[4, 0]], [30], [[1, 4, 9]], [3], 14, S)
    assert keep_tokens(*pool, i32([[4, 0]]), i32([30]), i32([[1, 4, 9]]), i32([3]), 14).tolist() == lengths
    assert all(torch.equal(a, b) for a, b in zip(pool, want))
    assert torch.equal(wide[:, :, 2], before[:, :, 2]) and torch.equal(wide[..., :4], before[..., :4])


def test_refused_trees_keep_their_history():
    pool = random_pool(4, 1, 2, 16, 64, 64, seed=2)
    before = [t.clone() for t in pool]
    for granted, want in ((0, [20]), (8, [14])):
        got = keep_tokens(*pool, i32([[0, 1]]), i32([20]), i32([[0, 5]]), i32([2]), 8, granted=i32([granted]))
        assert got.tolist() == want
        assert all(torch.equal(a, b) for a, b in zip(pool, before)) == (granted == 0)
    with pytest.raises(ValueError):
        keep_tokens(*pool, i32([[0, 1]]), i32([20]), i32([[0, 5]]), i32([2]), 8, granted=i32([1, 1]))
