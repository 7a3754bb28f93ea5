"""The operators of a speculative serving step over the packed cache, at the sizes it has them do.

A step drafts a tree of tokens per sequence, runs the model on all of them at once and keeps the
path that was accepted.  Around the model's own products that takes

  plan   block tables, slot maps, positions and tree masks from request lengths (`plan_tokens`)
  rope   norms of queries and keys for each head with the position rotation (`qk_norm_rope`)
  tree   attention of the drafted tokens over paged packed K/V (`tree_decode_attention`)
  keep   the accepted path's rows moved to the end of the kept history (`keep_tokens`)

`run` computes them in elementary torch operations, or with `own` by the package's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False                                  # set from outside: `run` then makes the package's calls

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _tree(name=None, *, batch, q_heads, kv_heads, drafted, lo, hi, page=16, bits_k=4, bits_v=4,
          dtype="bf16", head_dim=128, padded=0):
    """Histories log-uniform in [lo, hi]; `padded`: the last tokens of every second tree are padding."""
    c = {"name": name} if name else {}
    return {**c, "kind": "tree", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "drafted": drafted, "lo": lo, "hi": hi, "page": page, "bits_k": bits_k, "bits_v": bits_v,
            "dtype": dtype, "padded": padded}


def _rope(name=None, *, batch, tokens, q_heads, kv_heads, head_dim=128, rot=None, norm=True,
          interleaved=False, longest=8192, dtype="bf16", padded=0):
    c = {"name": name} if name else {}
    return {**c, "kind": "rope", "batch": batch, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rot": rot or head_dim, "norm": norm, "interleaved": interleaved,
            "longest": longest, "dtype": dtype, "padded": padded}


def _plan(name=None, *, batch, lo, hi, new_lo, new_hi, page=16, drafted=0):
    """`drafted` > 0: a tree of that many tokens per request, else new_lo .. new_hi tokens each."""
    c = {"name": name} if name else {}
    return {**c, "kind": "plan", "batch": batch, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi,
            "page": page, "drafted": drafted}


def _keep(name=None, *, batch, layers, kv_heads, drafted, accepted, lo, hi, page=16, bits_k=4, bits_v=4,
          head_dim=128):
    c = {"name": name} if name else {}
    return {**c, "kind": "keep", "batch": batch, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim,
            "drafted": drafted, "accepted": accepted, "lo": lo, "hi": hi, "page": page, "bits_k": bits_k,
            "bits_v": bits_v}


def listed():
    return [
        # one short chat on a small model, a handful of guesses in full precision: latency
        _tree("tree_b1_1k_fp32", batch=1, q_heads=8, kv_heads=2, drafted=8, lo=1000, hi=1000, dtype="fp32"),
        # a usual serving batch, every request with a tree of 32 tokens
        _tree("tree_b16_8k_q32", batch=16, q_heads=32, kv_heads=8, drafted=32, lo=8192, hi=8192),
        # one very long document, a wide tree
        _tree("tree_b1_128k_q64", batch=1, q_heads=64, kv_heads=8, drafted=64, lo=131072, hi=131072, page=64,
              dtype="fp16"),
        # a full server: all lengths, keys narrower than values, trees cut short by padding
        _tree("tree_b48_ragged_q13", batch=48, q_heads=32, kv_heads=8, drafted=13, lo=300, hi=16384, bits_v=6,
              padded=5),
        # a half-billion-parameter model: head_dim 64, seven query heads to a kv head
        _tree("tree_b8_d64_q24", batch=8, q_heads=14, kv_heads=2, drafted=24, lo=700, hi=5000, head_dim=64),
        # the smallest call: one token of a small model, rotation only
        _rope("rope_b1_token", batch=1, tokens=1, q_heads=14, kv_heads=2, head_dim=64, norm=False),
        # the drafted tokens of a batch
        _rope("rope_b32_q16", batch=32, tokens=16, q_heads=32, kv_heads=8, longest=32768, padded=3),
        # a long prompt in one piece, positions far out
        _rope("rope_prompt_8k", batch=1, tokens=8191, q_heads=32, kv_heads=8, longest=131072),
        # a verify step's tables, slots and masks
        _plan("plan_b32_tree32", batch=32, lo=100, hi=16384, new_lo=32, new_hi=32, drafted=32),
        # new requests' prompts and running requests side by side
        _plan("plan_b96_prompts", batch=96, lo=1, hi=8192, new_lo=1, new_hi=1500, page=32),
        # the accepted tokens of a small batch, eight layers
        _keep("keep_b8_layers8", batch=8, layers=8, kv_heads=4, drafted=16, accepted=3, lo=100, hi=900),
        # a full server after a step with long accepted paths
        _keep("keep_b64_layers28", batch=64, layers=28, kv_heads=8, drafted=32, accepted=7, lo=60, hi=600,
              bits_v=6),
    ]


# ---- drawn cases ---------------------------------------------------------------------------
WIDTHS = ((4, 4), (4, 4), (4, 6), (6, 6), (8, 8))
HEADS = ((8, 2), (16, 8), (28, 4), (32, 8), (64, 8))
MAX_TREE_FLOPS = {"fp32": 2.0e10, "fp16": 2.0e11, "bf16": 2.0e11}
MAX_TREE_TOKENS = 1 << 20               # cached token heads of one pass
MAX_POOL_BYTES = 4.0e8


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(("tree", "tree", "tree", "rope", "rope", "plan", "keep"))
    (bits_k, bits_v), (q_heads, kv_heads) = rng.choice(WIDTHS), rng.choice(HEADS)
    if kind == "tree":
        head_dim, dtype = 128, rng.choice(("bf16", "bf16", "fp16", "fp32"))
        if rng.random() < 0.2:                              # small models
            head_dim, q_heads, kv_heads = 64, 14, 2
        batch, drafted = _log(rng, 1, 64), _log(rng, 1, 96)
        room = min(MAX_TREE_TOKENS // (batch * kv_heads),
                   int(MAX_TREE_FLOPS[dtype] / (4.0 * batch * drafted * q_heads * head_dim)))
        hi = max(1, min(_log(rng, 50, 131072 if batch == 1 else 32768), room - drafted))
        lo = rng.choice((hi, max(1, hi // 8), max(1, hi // 64)))
        return _tree(batch=batch, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, drafted=drafted, lo=lo,
                     hi=hi, page=rng.choice((16, 16, 32, 64)), bits_k=bits_k, bits_v=bits_v, dtype=dtype,
                     padded=rng.choice((0, drafted // 3)))
    if kind == "rope":
        head_dim = rng.choice((64, 96, 128, 128, 256))
        batch = _log(rng, 1, 64)
        tokens = rng.choice((1, _log(rng, 2, 64), _log(rng, 65, 8191)))
        tokens = max(1, min(tokens, 8191 * 40 * 128 // (batch * (q_heads + kv_heads) * head_dim)))
        return _rope(batch=batch, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                     rot=rng.choice((head_dim, head_dim, head_dim // 2)), norm=rng.random() < 0.7,
                     interleaved=rng.random() < 0.3, longest=rng.choice((8192, 32768, 131072)),
                     dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), padded=rng.choice((0, tokens // 4)))
    if kind == "plan":
        batch, page = _log(rng, 1, 128), rng.choice((16, 32, 64))
        lo, hi = _log(rng, 1, 200), _log(rng, 201, 16384)
        if rng.random() < 0.5:
            drafted = _log(rng, 1, 96)
            return _plan(batch=batch, lo=lo, hi=hi, new_lo=drafted, new_hi=drafted, page=page, drafted=drafted)
        return _plan(batch=batch, lo=lo, hi=hi, new_lo=1, new_hi=rng.choice((1, _log(rng, 2, 1500))), page=page)
    layers, page, drafted = _log(rng, 1, 32), rng.choice((16, 32, 64)), _log(rng, 2, 64)
    per_token = layers * kv_heads * (128 * (bits_k + bits_v) // 8 + 4)
    batch = max(1, min(_log(rng, 1, 64), int(MAX_POOL_BYTES / (per_token * (drafted + 64 + 100)))))
    hi = max(1, min(_log(rng, 50, 2000), int(MAX_POOL_BYTES / (per_token * batch)) - drafted - 64))
    return _keep(batch=batch, layers=layers, kv_heads=kv_heads, drafted=drafted,
                 accepted=rng.randint(1, min(drafted, 12)), lo=max(1, hi // 8), hi=hi, page=page, bits_k=bits_k,
                 bits_v=bits_v)


# ---- inputs --------------------------------------------------------------------------------
def _spread(lo: int, hi: int, count: int) -> list[int]:
    """`count` lengths log-evenly spaced over [lo, hi]: their sum depends on the case alone."""
    return [int(round(math.exp(math.log(lo) + (math.log(hi) - math.log(lo)) * (i + 0.5) / count)))
            for i in range(count)]


def _shuffled(values, rng: random.Random):
    values = list(values)
    rng.shuffle(values)
    return values


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _parents(c, rng: random.Random) -> list[list[int]]:
    """Drafted trees, token 0 the root: each token hangs below one of the last few before it.
    Padding tokens (-2) are the last ones of every second tree."""
    rows = []
    for b in range(c["batch"]):
        real = c["drafted"] - (c.get("padded", 0) if b % 2 else 0)
        rows.append([-1 if i == 0 else i - 1 - rng.randrange(min(i, 5)) if i < real else -2
                     for i in range(c["drafted"])])
    return rows


def _reach(parents: torch.Tensor):
    """(B, Q) parents -> (B, Q, Q) bool: token i sees token j, its ancestor or itself; False for padding."""
    B, Q = parents.shape
    eye = torch.eye(Q, dtype=torch.float64, device=parents.device)
    step = (parents[..., None] == torch.arange(Q, device=parents.device)).double()
    reach = torch.linalg.solve_triangular(eye - step, eye.expand(B, Q, Q), upper=False, unitriangular=True) > 0.5
    return reach & (parents >= -1)[..., None]


def _words(reach: torch.Tensor) -> torch.Tensor:
    """(B, Q, Q) bool -> (B, Q, ceil(Q / 32)) int32, bit j % 32 of word j // 32 for token j."""
    B, Q = reach.shape[:2]
    W = -(-Q // 32)
    bits = torch.zeros(B, Q, 32 * W, dtype=torch.int64, device=reach.device)
    bits[..., :Q] = reach
    words = (bits.view(B, Q, W, 32) << torch.arange(32, device=reach.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _codebook(bits: int, head_dim: int) -> torch.Tensor:
    """Lloyd-Max levels of a coordinate of a random unit vector, N(0, 1 / head_dim), in 64 bits."""
    n = 1 << bits
    c = torch.special.ndtri((torch.arange(n, dtype=torch.float64) + 0.5) / n)
    for _ in range(60):
        edge = torch.cat([torch.tensor([-40.0], dtype=torch.float64), (c[1:] + c[:-1]) / 2,
                          torch.tensor([40.0], dtype=torch.float64)])
        density = torch.exp(-0.5 * edge * edge) / math.sqrt(2 * math.pi)
        mass = torch.special.ndtr(edge)
        c = (density[:-1] - density[1:]) / (mass[1:] - mass[:-1]).clamp_min(1e-300)
    return c / math.sqrt(head_dim)


def _pack(codes: torch.Tensor, bits: int) -> torch.Tensor:
    """(..., D) integer codes -> (..., D * bits / 8) uint8, least significant bits first."""
    x = codes.to(torch.int32)
    if bits == 8:
        return x.to(torch.uint8)
    if bits == 4:
        return (x[..., 0::2] | x[..., 1::2] << 4).to(torch.uint8)
    a, b, c, d = (x[..., i::4] for i in range(4))                     # 6 bits: four codes in three bytes
    word = a | b << 6 | c << 12 | d << 18
    return torch.stack([word & 255, word >> 8 & 255, word >> 16], -1).flatten(-2).to(torch.uint8)


def _rotation(head_dim: int, g) -> torch.Tensor:
    q, r = torch.linalg.qr(torch.randn(head_dim, head_dim, device="cuda", generator=g, dtype=torch.float64))
    return (q * torch.sign(torch.diagonal(r))).float().contiguous()


def _packed_pages(pages, heads, page, head_dim, bits, g):
    """Pages of codes of random vectors and their norms, the codebook and the rotation."""
    levels = _codebook(bits, head_dim).cuda()
    edges = ((levels[1:] + levels[:-1]) / 2).float()
    rows = pages * heads * page
    out = torch.empty(rows, head_dim * bits // 8, dtype=torch.uint8, device="cuda")
    for at in range(0, rows, 1 << 20):
        x = torch.randn(min(1 << 20, rows - at), head_dim, device="cuda", generator=g) / math.sqrt(head_dim)
        out[at:at + x.shape[0]] = _pack(torch.bucketize(x, edges, out_int32=True), bits)
    norms = (math.sqrt(head_dim) * torch.exp(0.3 * torch.randn(rows, device="cuda", generator=g))).half()
    return (out.view(pages, heads, page, -1), norms.view(pages, heads, page), levels.float().contiguous(),
            _rotation(head_dim, g))


def _table(lens, page, g, spare=0, width=None):
    """A random assignment of pages to sequences: (table, pages in the pool, pages left over)."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare, order[at:].contiguous()


def _prepare_tree(c, seed):
    g, rng = _generator(seed), random.Random(seed * 7919 + 13)
    hist = _shuffled(_spread(c["lo"], c["hi"], c["batch"]), rng)
    lens = [n + c["drafted"] for n in hist]
    table, pages, _ = _table(lens, c["page"], g)
    D, dtype = c["head_dim"], DTYPES[c["dtype"]]
    k_pages, k_norms, k_levels, k_rot = _packed_pages(pages, c["kv_heads"], c["page"], D, c["bits_k"], g)
    v_pages, v_norms, v_levels, v_rot = _packed_pages(pages, c["kv_heads"], c["page"], D, c["bits_v"], g)
    parents = torch.tensor(_parents(c, rng), dtype=torch.int32).cuda()
    # queries as a norm for each head leaves them: about sqrt(head_dim) long
    q = torch.randn(c["batch"], c["drafted"], c["q_heads"], D, device="cuda", generator=g).to(dtype)
    s = {"kind": "tree", "q": q.transpose(1, 2), "k_pages": k_pages, "k_norms": k_norms, "v_pages": v_pages,
         "v_norms": v_norms, "table": table, "seq_lens": torch.tensor(lens, dtype=torch.int32).cuda(),
         "k_levels": k_levels, "v_levels": v_levels, "k_rot": k_rot, "v_rot": v_rot, "bits_k": c["bits_k"],
         "bits_v": c["bits_v"], "mask": _words(_reach(parents)), "scale": D ** -0.5}
    if own:                                  # the layer's handle, which a serving program keeps
        from winnow_b200 import packed_attention as pa
        s["kv"] = pa.PackedKV(k_pages, k_norms, v_pages, v_norms, table, s["seq_lens"],
                              pa.Quantizer(k_rot, k_levels, c["bits_k"]),
                              pa.Quantizer(v_rot, v_levels, c["bits_v"]), D)
    return s


def _prepare_rope(c, seed):
    g, rng = _generator(seed), random.Random(seed * 7919 + 13)
    B, n, D, dtype = c["batch"], c["tokens"], c["head_dim"], DTYPES[c["dtype"]]
    heads = c["q_heads"] + 2 * c["kv_heads"]
    # what the fused projection of a layer leaves: queries, keys and values of a token side by side
    qkv = (2.0 * torch.randn(B, n, heads, D, device="cuda", generator=g)).to(dtype)
    start = torch.tensor([rng.randrange(max(1, c["longest"] - n)) for _ in range(B)])
    positions = start[:, None] + torch.arange(n)[None]
    if c["padded"]:
        positions[1::2, n - c["padded"]:] = -1
    angle = torch.arange(c["longest"], dtype=torch.float64, device="cuda")[:, None] \
        * 1e6 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    weights = [(1.0 + 0.2 * torch.randn(D, device="cuda", generator=g)).to(dtype) if c["norm"] else None
               for _ in range(2)]
    return {"kind": "rope", "q": qkv[:, :, :c["q_heads"]].transpose(1, 2),
            "k": qkv[:, :, c["q_heads"]:c["q_heads"] + c["kv_heads"]].transpose(1, 2),
            "positions": positions.to(torch.int32).cuda(),
            "table": torch.cat([angle.cos(), angle.sin()], -1).float(), "q_weight": weights[0],
            "k_weight": weights[1], "eps": 1e-6, "interleaved": c["interleaved"]}


def _prepare_plan(c, seed):
    g, rng = _generator(seed), random.Random(seed * 7919 + 13)
    B, S = c["batch"], c["page"]
    hist = _shuffled(_spread(c["lo"], c["hi"], B), rng)
    new = _shuffled(_spread(c["new_lo"], c["new_hi"], B), rng)
    grow = sum(-(-(h + n) // S) - -(-h // S) for h, n in zip(hist, new))
    width = -(-(c["hi"] + c["new_hi"]) // S) + 1
    table, _, free = _table(hist, S, g, spare=grow + 64, width=width)
    as_int = lambda v: torch.tensor(v, dtype=torch.int32).cuda()       # noqa: E731
    return {"kind": "plan", "lengths": as_int(hist), "new": None if c["drafted"] else as_int(new),
            "parents": as_int(_parents(c, rng)) if c["drafted"] else None, "table": table,
            "held": as_int([-(-h // S) for h in hist]), "free": free, "free_count": as_int([free.numel()]),
            "page": S, "tokens": sum(new)}


def _prepare_keep(c, seed):
    g, rng = _generator(seed), random.Random(seed * 7919 + 13)
    lens = [n + c["drafted"] for n in _shuffled(_spread(c["lo"], c["hi"], c["batch"]), rng)]
    table, pages, _ = _table(lens, c["page"], g)
    lead = (c["layers"], pages, c["kv_heads"], c["page"])
    s = {"kind": "keep", "table": table, "seq_lens": torch.tensor(lens, dtype=torch.int32).cuda(),
         "drafted": c["drafted"]}
    for side in "kv":
        nb = c["head_dim"] * c["bits_" + side] // 8
        s[side + "_pages"] = torch.randint(0, 256, (*lead, nb), dtype=torch.uint8, device="cuda", generator=g)
        s[side + "_norms"] = (5 + 20 * torch.rand(lead, device="cuda", generator=g)).half()
    # accepted paths: the root, then later and later tokens; the places behind a path hold nothing
    paths = [[0] + sorted(rng.sample(range(1, c["drafted"]), c["accepted"] - 1)) for _ in range(c["batch"])]
    s["keep"] = torch.tensor([p + [-1, -1] for p in paths], dtype=torch.int32).cuda()
    s["counts"] = torch.full((c["batch"],), c["accepted"], dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    return {"tree": _prepare_tree, "rope": _prepare_rope, "plan": _prepare_plan,
            "keep": _prepare_keep}[case["kind"]](dict(case), seed)


# ---- plain forms ---------------------------------------------------------------------------
def _codes(rows: torch.Tensor, bits: int) -> torch.Tensor:
    """(..., D * bits / 8) uint8 -> (..., D) int32 codes."""
    nb = rows.shape[-1]
    bit = torch.arange(nb * 8 // bits, device=rows.device) * bits
    low, high = rows[..., bit >> 3].to(torch.int32), rows[..., ((bit >> 3) + 1).clamp_max(nb - 1)].to(torch.int32)
    return (low | high << 8) >> (bit & 7).to(torch.int32) & (1 << bits) - 1


def _history(pages, norms, table, levels, bits):
    """Every sequence's rows in the quantizer's basis, norms applied: (B, Hkv, W * S, D) fp32."""
    at = table.clamp_min(0).long()
    rows = levels[_codes(pages[at], bits).long()] * norms[at].float()[..., None]        # (B, W, Hkv, S, D)
    return rows.transpose(1, 2).flatten(2, 3)


def _visible(seq_lens, mask, drafted, width):
    """(B, Q, width) bool: the history for every token that is not padding, and the tree by its bits."""
    at = torch.arange(width, device=mask.device)[None] - (seq_lens - drafted)[:, None]  # (B, T): place in the tree
    inside = (at >= 0) & (at < drafted)
    j = at.clamp(0, drafted - 1).long()
    word = torch.gather(mask, 2, (j >> 5)[:, None].expand(-1, drafted, -1))
    seen = (word >> (j & 31).to(torch.int32)[:, None]) & 1
    real = (mask != 0).any(-1)[..., None]
    return (at < 0)[:, None] & real | inside[:, None] & (seen != 0)


def _plain_tree(s):
    q = s["q"].float()
    B, Hq, Q, D = q.shape
    keys = _history(s["k_pages"], s["k_norms"], s["table"], s["k_levels"], s["bits_k"])
    values = _history(s["v_pages"], s["v_norms"], s["table"], s["v_levels"], s["bits_v"])
    Hkv, T = keys.shape[1:3]
    rows = (q @ s["k_rot"].T * s["scale"]).reshape(B, Hkv, -1, D)                       # rows (head, token)
    scores = (rows @ keys.transpose(-1, -2)).view(B, Hq, Q, T)
    scores = scores.masked_fill(~_visible(s["seq_lens"], s["mask"], Q, T)[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, Hkv, -1, T) @ values).view(B, Hq, Q, D) @ s["v_rot"]
    return torch.where(total > 0, out / total.clamp_min(1e-30), 0.0).to(s["q"].dtype)


def _plain_rope_of(x, weight, s):
    y, rot = x.float(), s["table"].shape[1]
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * weight.float()
    turn = s["table"][s["positions"].clamp_min(0).long()][:, None]                       # (B, 1, n, rot)
    cos, sin = turn[..., :rot // 2], turn[..., rot // 2:]
    if s["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    out = torch.cat([turned, y[..., rot:]], -1)
    return torch.where((s["positions"] >= 0)[:, None, :, None], out, 0.0).to(x.dtype)


def _plain_plan(s):
    lengths, table, page, T = s["lengths"], s["table"], s["page"], s["tokens"]
    B, W = table.shape
    tree = s["parents"] is not None
    new = torch.full_like(lengths, T // B) if tree else s["new"]
    after = lengths + new
    held = torch.maximum(s["held"], (after + page - 1) // page)
    grow = held - s["held"]
    taken = torch.cumsum(grow, 0, dtype=torch.int32)
    column = torch.arange(W, device=table.device, dtype=torch.int32)[None]
    fresh = (column >= s["held"][:, None]) & (column < held[:, None])
    stack = s["free_count"] - 1 - ((taken - grow)[:, None] + column - s["held"][:, None])
    table.copy_(torch.where(fresh, s["free"][stack.clamp(0, s["free"].numel() - 1).long()], table))
    starts = torch.cat([torch.zeros_like(taken[:1]), torch.cumsum(new, 0, dtype=torch.int32)])
    token = torch.arange(T, device=table.device, dtype=torch.int32)
    sequence = torch.searchsorted(starts[1:], token, right=True).to(torch.int32)
    b = sequence.long()
    at = lengths[b] + token - starts[b]
    out = {"table": table, "seq_lens": after, "held": held, "free_count": s["free_count"] - taken[-1:],
           "starts": starts, "sequence": sequence, "positions": at,
           "slot_pages": table[b, (at // page).long()][:, None], "slot_ends": at % page + 1}
    if tree:
        reach = _reach(s["parents"])
        depth = reach.sum(-1, dtype=torch.int32) - 1
        out["positions"] = torch.where(depth >= 0, lengths[:, None] + depth, -1).flatten()
        out["mask"] = _words(reach)
    return out


def _plain_keep(s):
    base = s["seq_lens"] - s["drafted"]
    page, A = s["k_norms"].shape[3], s["keep"].shape[1]
    i = torch.arange(A, device=base.device)[None]
    moved = i < s["counts"][:, None]
    source, target = (base[:, None] + s["keep"])[moved], (base[:, None] + i)[moved]
    b = torch.arange(base.numel(), device=base.device)[:, None].expand(-1, A)[moved]
    from_page, to_page = (s["table"][b, (t // page).long()].long() for t in (source, target))
    from_slot, to_slot = (source % page).long(), (target % page).long()
    pool = [s[name] for name in ("k_pages", "k_norms", "v_pages", "v_norms")]
    rows = [x[:, from_page, :, from_slot] for x in pool]                 # read before anything is written
    pool[0][:, to_page, :, to_slot] = rows[0]
    pool[1][:, to_page, :, to_slot] = rows[1]
    pool[2][:, to_page, :, to_slot] = rows[2]
    pool[3][:, to_page, :, to_slot] = rows[3]
    return base + s["counts"]


# ---- one pass ------------------------------------------------------------------------------
def _own_tree(s):
    from winnow_b200.packed_attention_cuda import tree_decode_attention
    return tree_decode_attention(s["q"], s["kv"], s["mask"], s["scale"], check_page_ids=False)


def _own_rope(s):
    from winnow_b200.rotary import qk_norm_rope
    return qk_norm_rope(s["q"], s["k"], s["positions"], s["table"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                        eps=s["eps"], interleaved=s["interleaved"])


def _own_plan(s):
    from winnow_b200.block_tables import plan_tokens
    p = plan_tokens(s["lengths"], s["new"], s["table"], s["held"], s["free"], s["free_count"], s["page"],
                    s["tokens"], parents=s["parents"])
    out = {"table": s["table"], "seq_lens": p.seq_lens, "held": p.held, "free_count": p.free_count,
           "starts": p.starts, "sequence": p.sequence, "positions": p.positions, "slot_pages": p.slot_pages,
           "slot_ends": p.slot_ends}
    return out if p.mask is None else {**out, "mask": p.mask}


def _own_keep(s):
    from winnow_b200.packed_backend import keep_tokens
    return keep_tokens(s["k_pages"], s["k_norms"], s["v_pages"], s["v_norms"], s["table"], s["seq_lens"],
                       s["keep"], s["counts"], s["drafted"])


def run(s):
    kind = s["kind"]
    if kind == "tree":
        return _own_tree(s) if own else _plain_tree(s)
    if kind == "rope":
        return _own_rope(s) if own else (_plain_rope_of(s["q"], s["q_weight"], s),
                                         _plain_rope_of(s["k"], s["k_weight"], s))
    if kind == "plan":
        return _own_plan(s) if own else _plain_plan(s)
    lengths = _own_keep(s) if own else _plain_keep(s)
    return [lengths, s["k_pages"], s["k_norms"], s["v_pages"], s["v_norms"]]


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    c = dict(case)
    if c["kind"] == "tree":
        el = DTYPES[c["dtype"]].itemsize
        hist = _spread(c["lo"], c["hi"], c["batch"])
        tokens, Q, D = sum(hist) + c["batch"] * c["drafted"], c["drafted"], c["head_dim"]
        row = D * (c["bits_k"] + c["bits_v"]) // 8 + 4
        real = sum(Q - (c["padded"] if b % 2 else 0) for b in range(c["batch"])) / c["batch"]   # of a tree
        # each real token scores and sums the history and, on average, a few tokens of its tree
        return {"bytes": tokens * c["kv_heads"] * row + 4 * tokens // c["page"]
                + c["batch"] * Q * (2 * c["q_heads"] * D * el + 4 * -(-Q // 32)),
                "flops": 4.0 * sum(hist) * real * c["q_heads"] * D}
    if c["kind"] == "rope":
        el, tokens = DTYPES[c["dtype"]].itemsize, c["batch"] * c["tokens"]
        values = tokens * (c["q_heads"] + c["kv_heads"]) * c["head_dim"]
        return {"bytes": 2 * values * el + tokens * (4 + 4 * c["rot"]), "flops": (7.0 if c["norm"] else 3.0) * values}
    if c["kind"] == "plan":
        hist, new = (_spread(c[a], c[b], c["batch"]) for a, b in (("lo", "hi"), ("new_lo", "new_hi")))
        tokens, Q, S = sum(new), c["drafted"], c["page"]
        pages = tokens // S + c["batch"]                     # table entries read or written
        return {"bytes": 24 * c["batch"] + 16 * tokens + 8 * pages + (4 + 4 * -(-Q // 32)) * c["batch"] * Q,
                "flops": 0.0}
    moved = c["batch"] * (c["accepted"] - 1)                 # the root stays where it is
    row = c["head_dim"] * (c["bits_k"] + c["bits_v"]) // 8 + 4
    return {"bytes": 2 * moved * c["layers"] * c["kv_heads"] * row + 20 * c["batch"] + 8 * c["batch"] * c["accepted"],
            "flops": 0.0}


# ---- the definitions in 64 bits ------------------------------------------------------------
def _exact_tree(s, c):
    """Reconstruct keys and values row by row in the model's basis, then softmax over what is seen."""
    B, Hq, Q, D = s["q"].shape
    out = torch.zeros(B, Hq, Q, D, dtype=torch.float64, device="cuda")
    group = Hq // c["kv_heads"]
    shift = torch.arange(32, device="cuda", dtype=torch.int32)
    tree = ((s["mask"][..., None] >> shift) & 1).flatten(-2)[..., :Q].bool()             # (B, Q, Q)
    for b in range(B):
        L = int(s["seq_lens"][b])
        ids = s["table"][b, :-(-L // c["page"])].long()
        seen = torch.ones(Q, L, dtype=torch.bool, device="cuda")
        seen[:, L - Q:] = tree[b]
        seen &= tree[b].any(-1, keepdim=True)
        for h in range(c["kv_heads"]):
            kv = []
            for side in "kv":
                rows, bits = s[side + "_pages"][ids, h].flatten(0, 1)[:L], c["bits_" + side]
                stream = (rows[..., None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
                bit = stream.flatten(-2).view(L, D, bits).long()
                code = (bit << torch.arange(bits, device="cuda")).sum(-1)
                unit = s[side + "_levels"].double()[code] @ s[side + "_rot"].double()
                kv.append(unit * s[side + "_norms"][ids, h].flatten()[:L].double()[:, None])
            heads = s["q"][b, h * group:(h + 1) * group].double()
            score = (heads @ kv[0].T) * s["scale"]
            score = torch.where(seen, score, -torch.inf)
            p = torch.nan_to_num(torch.softmax(score, -1), nan=0.0)
            out[b, h * group:(h + 1) * group] = p @ kv[1]
    return out


def _exact_rope_of(x, weight, s):
    y = x.double()
    if weight is not None:
        y = y / (y.square().sum(-1, keepdim=True) / y.shape[-1] + s["eps"]).sqrt() * weight.double()
    rot = s["table"].shape[1]
    turn = s["table"].double()[s["positions"].long().clamp_min(0)].unsqueeze(1)
    turn = torch.complex(turn[..., :rot // 2].contiguous(), turn[..., rot // 2:].contiguous())
    pairs = y[..., :rot]
    pairs = pairs.unflatten(-1, (rot // 2, 2)) if s["interleaved"] else pairs.unflatten(-1, (2, rot // 2)).mT
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y = torch.cat([turned.flatten(-2) if s["interleaved"] else turned.mT.flatten(-2), y[..., rot:]], -1)
    y[(s["positions"] < 0)[:, None].expand(y.shape[:-1])] = 0.0
    return y


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "plan":
        return None                                          # whole numbers only
    s = prepare(c, seed)
    if c["kind"] == "tree":
        return _exact_tree(s, c)
    if c["kind"] == "rope":
        return _exact_rope_of(s["q"], s["q_weight"], s), _exact_rope_of(s["k"], s["k_weight"], s)
    norms = []
    table, keep = s["table"].cpu(), s["keep"].cpu()
    for x in (s["k_norms"], s["v_norms"]):                   # norms are numbers: moved one by one
        y = x.double()
        for b, L in enumerate(s["seq_lens"].tolist()):
            for i in range(c["accepted"]):
                a, z = L - c["drafted"] + int(keep[b, i]), L - c["drafted"] + i
                y[:, table[b, z // c["page"]], :, z % c["page"]] = \
                    x[:, table[b, a // c["page"]], :, a % c["page"]].double()
        norms.append(y)
    return [None, None, norms[0], None, norms[1]]
