"""Norms of queries and keys for each head with the rotary position rotation, in one pass.

What a model's attention layer does to its fused projection's output before the
cache's append and the attention (the reference leaves it to Transformers'
modelling code): every head's row is normalised (optionally) and turned by its
token's position, in fp32 with one rounding, straight from the projection's
strided output into the tensors the next calls read (`wtq_qk_norm_rope`).
Inference only, like the rest of the package: there is no backward pass, and tensors that
carry tangents are refused.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib


@dataclass
class Rotary:
    """A model's position rotation, with the norms of its layers' queries and keys where it has them:
    `q_weights[i]`, `k_weights[i]` (D,) of layer i, or None for no norm."""

    table: torch.Tensor
    q_weights: list | None = None
    k_weights: list | None = None
    eps: float = 1e-6
    interleaved: bool = False

    def apply(self, layer: int, q, k, positions, *, v=None, out=None, status=None):
        """`qk_norm_rope` with what layer `layer` has."""
        return qk_norm_rope(q, k, positions, self.table, eps=self.eps, interleaved=self.interleaved, v=v, out=out,
                            q_weight=None if self.q_weights is None else self.q_weights[layer],
                            k_weight=None if self.k_weights is None else self.k_weights[layer], status=status)


def rotary_table(rot: int, positions: int, *, base: float = 10000.0, inv_freq: torch.Tensor | None = None,
                 scale: float = 1.0, device="cuda") -> torch.Tensor:
    """(positions, rot) fp32: the cosines of a position's rot / 2 pairs, then their sines, times `scale`.
    Angles are position * inv_freq (base ** (-2 i / rot) when not given) in 64 bits: in 32, an angle of
    100 000 turns would be off by thousandths."""
    if rot < 2 or rot % 2:
        raise ValueError(f"rot must be even and positive, got {rot}")
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    if inv_freq.numel() != rot // 2:
        raise ValueError(f"inv_freq needs {rot // 2} entries, got {inv_freq.numel()}")
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] \
        * inv_freq.to(device, torch.float64).reshape(1, -1)
    return (torch.cat([angle.cos(), angle.sin()], -1) * scale).float().contiguous()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = False, v: torch.Tensor | None = None, out=None,
                 status: torch.Tensor | None = None):
    """q (B, Hq, n, D), k (B, Hkv, n, D) -> the pair normalised and turned, in their dtype.

    q, k (and v) are CUDA tensors of one float type, any strides with a contiguous last dimension (slices
    of a fused projection as they are).  `positions` (B, n) int32; a negative one is padding, whose
    queries and keys become zeros, and so does one that `table` does not have, which also sets
    `STATUS_BAD_POSITION` in `status`.  `table`: `rotary_table`'s, (rows, rot) with rot <= D; the
    coordinates past rot are not turned.  Pairs are (i, i + rot / 2), or (2 i, 2 i + 1) with
    `interleaved`.  A side with a weight (D,) is divided by the root of its mean square (plus `eps`) and
    multiplied by the weight first.  With `v` the values are copied along and the result has three
    tensors.  `out`: tensors of the same shapes to write into; they may be the inputs themselves, unless those
    are broadcast.
    """
    got = _lib.host().rope(q, k, v, positions, table, q_weight, k_weight, float(eps), interleaved,
                           out if out is None else tuple(out), status)      # checked and launched in native code
    if got is not None:
        return got
    xs = [q, k] if v is None else [q, k, v]
    weights = [q_weight, k_weight]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*xs, *weights, table)):
        raise RuntimeError("qk_norm_rope has no backward pass: call it under torch.no_grad()")
    _lib.no_tangents("qk_norm_rope", *xs, *weights, table)
    dev = _lib.require_cuda(*xs, positions, table, *(w for w in weights if w is not None))
    _lib.reachable("status", status, dev)
    if any(t.dim() != 4 for t in xs) or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:] \
            or (v is not None and v.shape != k.shape):
        raise ValueError("q must be (B, Hq, n, D), k and v (B, Hkv, n, D)")
    B, _, n, D = q.shape
    code = _lib.dtype_code(q.dtype)
    if any(t.dtype != q.dtype for t in xs):
        raise ValueError("q, k and v must have one dtype")
    if tuple(positions.shape) != (B, n) or positions.dtype != torch.int32:
        raise ValueError(f"positions must be int32 ({B}, {n})")
    if table.dim() != 2 or table.dtype != torch.float32 or table.stride(1) != 1 or table.shape[1] > D \
            or table.shape[1] % 2:
        raise ValueError("table must be fp32 (positions, rot) with contiguous rows and an even rot <= D")
    given = [w for w in weights if w is not None]
    if any(tuple(w.shape) != (D,) or not w.is_contiguous() or w.dtype != given[0].dtype for w in given):
        raise ValueError(f"weights must be contiguous ({D},) tensors of one dtype")
    with torch.no_grad():
        xs = [t if t.stride(-1) == 1 or D == 1 else t.contiguous() for t in xs]
        if positions.stride(-1) != 1 and n > 1:
            positions = positions.contiguous()
    if out is None:
        outs = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in xs]
    else:
        outs = list(out)
        if len(outs) != len(xs) or any(o.shape != t.shape or o.dtype != t.dtype or o.device != dev
                                       or (o.stride(-1) != 1 and D > 1) for o, t in zip(outs, xs)):
            raise ValueError("out needs a tensor of each input's shape and dtype with a contiguous last dimension")
        if any(_meets_itself(o) for o in outs):            # (several blocks would write, or turn in place, the same memory)
            raise ValueError("the tensors of out must not overlap themselves")
        for i, o in enumerate(outs):
            for j, t in enumerate(xs):
                same = i == j and o.data_ptr() == t.data_ptr() and o.stride() == t.stride()
                if not same and _lib.overlaps(o, t) and not _interleaved_slices(o, t):
                    raise ValueError("out may be the inputs themselves, but must not overlap them in another way")
            if any(_lib.overlaps(o, t) and not _interleaved_slices(o, t) for t in outs[:i]):
                raise ValueError("the tensors of out must not overlap")
    sides = (_lib.RopeSide * 3)()
    for i, (x, o) in enumerate(zip(xs, outs)):
        w = weights[i] if i < 2 else None
        sides[i] = _lib.RopeSide(x.data_ptr(), o.data_ptr(), _lib.i64x(*x.stride()[:3]), _lib.i64x(*o.stride()[:3]),
                                 None if w is None else w.data_ptr(), x.shape[1])
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().wtq_qk_norm_rope(
            sides, code, _lib.dtype_code(given[0].dtype) if given else code, float(eps), positions.data_ptr(),
            positions.stride(0), table.data_ptr(), table.stride(0), table.shape[0], B, n, D, table.shape[1],
            int(bool(interleaved)), None if status is None else status.data_ptr(), _lib.stream_ptr(dev)))
    return tuple(outs)


def _meets_itself(t: torch.Tensor) -> bool:
    """Whether two places of a tensor are one element, as in a broadcast one (strides that nest do not meet)."""
    reach = 1
    for step, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if step < reach:
            return t.numel() > 0
        reach = step * (n - 1) + reach
    return False


def _interleaved_slices(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two head ranges of one (B, n, heads, D) buffer: their ranges of addresses meet, their elements do
    not.  Both have the buffer's strides, so the distance between them is whole heads apart."""
    if a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() or a.stride() != b.stride():
        return False
    batch, step, token = a.stride()[:3]
    off = b.storage_offset() - a.storage_offset()
    if step < max(1, a.shape[3]) or off % step or token % step or token < 1 or batch % token:
        return False
    first, room = off // step, token // step               # heads from a's first to b's first; heads of a token
    low, high = (a, b) if first > 0 else (b, a)
    return low.shape[1] <= abs(first) and abs(first) + high.shape[1] <= room
