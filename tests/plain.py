"""The operators of a drafted step from their definitions, in 64 bits or whole numbers, on any device."""
from __future__ import annotations

import torch


def reach(parents):
    """(B, Q) nested list or tensor of parents -> (B, Q, Q) bool, walked token by token."""
    rows = parents.tolist() if isinstance(parents, torch.Tensor) else parents
    B, Q = len(rows), len(rows[0])
    seen = torch.zeros(B, Q, Q, dtype=torch.bool)
    for b, row in enumerate(rows):
        for i in range(Q):
            path, j = [], i
            while j >= 0:
                path.append(j)
                j = row[j] if -2 <= row[j] < j else -2
            if j == -1:
                seen[b, i, path] = True
    return seen


def words(seen):
    """(B, Q, Q) bool -> (B, Q, ceil(Q / 32)) int32."""
    B, Q = seen.shape[:2]
    out = torch.zeros(B, Q, -(-Q // 32), dtype=torch.int64)
    for j in range(Q):
        out[:, :, j // 32] |= seen[:, :, j].cpu().long() << (j % 32)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


def dequantised(pages, norms, quant, table, L, S, D):
    """(Hkv, L, D) rows of a sequence in 64 bits, page ids outside the pool read as zeros."""
    ids = table[: -(-L // S)].long()
    good = (ids >= 0) & (ids < pages.shape[0])
    at = ids.clamp(0, pages.shape[0] - 1)
    rows = pages[at].permute(1, 0, 2, 3).flatten(1, 2)[:, :L]
    n = (norms[at].double() * good[:, None, None]).permute(1, 0, 2).flatten(1)[:, :L]
    bw = quant.bit_width
    bits = ((rows[..., None] >> torch.arange(8, device=rows.device, dtype=torch.uint8)) & 1).flatten(-2)
    code = (bits.view(*rows.shape[:2], D, bw).long() << torch.arange(bw, device=rows.device)).sum(-1)
    return (quant.centroids.double()[code] @ quant.Pi.double()) * n[..., None]


def tree_attention(q, kv, seen, scale):
    """(B, Hq, Q, D) in 64 bits; `seen` (B, Q, Q) bool.  A token that sees no tree token is padding: zeros."""
    B, Hq, Q, D = q.shape
    out = torch.zeros(B, Hq, Q, D, dtype=torch.float64, device=q.device)
    group = Hq // kv.num_kv_heads
    seen = seen.to(q.device)
    for b in range(B):
        L = int(kv.seq_lens[b])
        if L <= 0:
            continue
        k = dequantised(kv.k_pages, kv.k_norms, kv.k_quant, kv.page_table[b], L, kv.page_size, D)
        v = dequantised(kv.v_pages, kv.v_norms, kv.v_quant, kv.page_table[b], L, kv.page_size, D)
        hist = L - Q
        allowed = torch.ones(Q, L, dtype=torch.bool, device=q.device)
        allowed[:, max(hist, 0):] = seen[b][:, max(-hist, 0):]
        allowed &= seen[b].any(-1, keepdim=True)
        for h in range(kv.num_kv_heads):
            s = q[b, h * group:(h + 1) * group].double() @ k[h].T * scale
            s = s.masked_fill(~allowed, -torch.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            out[b, h * group:(h + 1) * group] = p @ v[h]
    return out


def norm_rope(x, positions, table, weight, eps, interleaved, turned=True):
    """(B, H, n, D) in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight.double()
    if not turned:
        return y
    rot = table.shape[1]
    row = table.double()[positions.long().clamp(0, table.shape[0] - 1)][:, None]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    pair = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out = y.clone()
    out[..., pair[0]] = y[..., pair[0]] * c - y[..., pair[1]] * s
    out[..., pair[1]] = y[..., pair[1]] * c + y[..., pair[0]] * s
    out[((positions < 0) | (positions >= table.shape[0]))[:, None].expand(out.shape[:-1])] = 0
    return out


def plan(lengths, new, table, held, free, count, S, tokens, parents=None):
    """One step on lists; returns a dict of lists (table rows changed in place), or None when refused."""
    B, W = len(lengths), len(table[0]) if table else 0
    Q = len(parents[0]) if parents else 0
    if parents:
        new = [Q] * B
    need = [-(-(L + n) // S) for L, n in zip(lengths, new)]
    grow = [max(0, n - h) for n, h in zip(need, held)]
    if sum(grow) > count or any(n > W for n in need) or sum(new) > tokens:
        return None
    starts, sequence, positions, pages, ends, top = [0], [], [], [], [], count
    for b in range(B):
        for c in range(held[b], held[b] + grow[b]):
            top -= 1
            table[b][c] = free[top]
        seen = reach([parents[b]])[0] if parents else None
        for i in range(new[b]):
            at = lengths[b] + i
            sequence.append(b)
            depth = int(seen[i].sum()) - 1 if parents else i
            positions.append(lengths[b] + depth if depth >= 0 else -1)
            pages.append(table[b][at // S])
            ends.append(at % S + 1)
        starts.append(starts[-1] + new[b])
    pad = [-1] * (tokens - starts[-1])
    return {"seq_lens": [L + n for L, n in zip(lengths, new)], "held": [h + g for h, g in zip(held, grow)],
            "free_count": [top], "starts": starts, "sequence": sequence + pad, "positions": positions + pad,
            "slot_pages": pages + pad, "slot_ends": ends + [0] * len(pad)}


def keep(pool, table, lens, paths, counts, drafted, S):
    """The four pool tensors with the kept rows moved, one by one in order, and the new lengths."""
    pool = [t.clone() for t in pool]
    out = []
    for b, L in enumerate(lens):
        base = L - drafted
        for i in range(counts[b]):
            src, dst = base + paths[b][i], base + i
            for t in pool:
                t[:, table[b][dst // S], :, dst % S] = t[:, table[b][src // S], :, src % S].clone()
        out.append(base + counts[b])
    return pool, out
