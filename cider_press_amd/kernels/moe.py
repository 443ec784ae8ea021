"""Routed experts around gather_qmm: router top-k, the sort of (token, slot)
rows by expert that gather_qmm's sorted form takes, and the weighted combine.

No reference counterpart: the reference names this as its unbuilt MoE
feature (docs/inference/feed-forward.md:98-107, 131-137).  Semantics are
stated in include/cpq.h (cpq_moe_route, cpq_moe_route_grouped, cpq_moe_combine).
"""
from __future__ import annotations

import struct

from .. import _lib
from . import Buffer, Commands, _ptr


def _check_route(op: str, logits: Buffer, tokens: int, n_experts: int, top_k: int, experts: Buffer, scores: Buffer,
                 lhs: Buffer, rhs: Buffer, inv: Buffer, offsets: Buffer) -> None:
    for b, dt in ((experts, "u32"), (scores, "f32"), (lhs, "u32"), (rhs, "u32"), (inv, "u32"), (offsets, "u32")):
        if b.dtype != dt:
            raise TypeError(f"{op}: expected a {dt} buffer, got {b.dtype}")
    rows = tokens * top_k
    for b in (experts, scores, lhs, rhs, inv):
        if len(b) < rows:
            raise _lib.InvalidArgument(f"{op}: an output buffer is shorter than tokens*top_k")
    if len(offsets) < n_experts + 1 or len(logits) < tokens * n_experts:
        raise _lib.InvalidArgument(f"{op}: offsets or logits buffer too short")


def moe_route(commands: Commands, logits: Buffer, tokens: int, n_experts: int, top_k: int, normalize: bool,
              experts: Buffer, scores: Buffer, lhs: Buffer, rhs: Buffer, inv: Buffer, offsets: Buffer) -> None:
    """Softmax top-k per token, then the stable sort of the tokens*top_k rows
    by expert.  experts/lhs/rhs/inv: u32 [tokens*top_k]; scores: f32
    [tokens*top_k]; offsets: u32 [n_experts + 1].  Encodes only."""
    _check_route("moe_route", logits, tokens, n_experts, top_k, experts, scores, lhs, rhs, inv, offsets)
    _lib.check(_lib.lib().cpq_moe_route(
        commands.handle, _lib.DTYPES[logits.dtype], _ptr(logits), tokens, n_experts, top_k, int(bool(normalize)),
        _ptr(experts), _ptr(scores), _ptr(lhs), _ptr(rhs), _ptr(inv), _ptr(offsets)))


# cpq_moe_router, packed.
_ROUTER = struct.Struct("@iPIIIif0P")


def _router(sigmoid, bias, n_groups, top_groups, group_best, normalize, scale) -> bytes:
    try:
        return _ROUTER.pack(bool(sigmoid), _ptr(bias) or 0, n_groups, top_groups, group_best, bool(normalize), scale)
    except (struct.error, OverflowError) as e:
        raise _lib.InvalidArgument(f"moe_route_grouped: {e}") from None


def moe_route_grouped(commands: Commands, logits: Buffer, tokens: int, n_experts: int, top_k: int, normalize: bool,
                      experts: Buffer, scores: Buffer, lhs: Buffer, rhs: Buffer, inv: Buffer, offsets: Buffer,
                      sigmoid: bool = False, bias=None, n_groups: int = 1, top_groups: int = 1, group_best: int = 1,
                      scale: float = 1.0) -> None:
    """moe_route with sigmoid scores, a bias (f32 [n_experts]) that only the
    choice sees, experts of the best groups only, and weights times scale.
    Encodes only."""
    _check_route("moe_route_grouped", logits, tokens, n_experts, top_k, experts, scores, lhs, rhs, inv, offsets)
    if bias is not None:
        if bias.dtype != "f32":
            raise TypeError(f"moe_route_grouped: expected a f32 buffer, got {bias.dtype}")
        if len(bias) < n_experts:
            raise _lib.InvalidArgument("moe_route_grouped: bias buffer too short")
    router = _router(sigmoid, bias, n_groups, top_groups, group_best, normalize, scale)
    _lib.check(_lib.lib().cpq_moe_route_grouped(
        commands.handle, _lib.DTYPES[logits.dtype], _ptr(logits), tokens, n_experts, top_k, router, _ptr(experts),
        _ptr(scores), _ptr(lhs), _ptr(rhs), _ptr(inv), _ptr(offsets)))


def moe_combine(commands: Commands, y: Buffer, scores: Buffer, inv: Buffer, tokens: int, top_k: int, n: int,
                out: Buffer) -> None:
    """out[t, :] = sum_j scores[t*k + j] * y[inv[t*k + j], :] (fp32, rounded to
    T); y holds the expert outputs in sorted row order.  Encodes only."""
    if scores.dtype != "f32" or inv.dtype != "u32":
        raise TypeError("moe_combine: scores must be f32 and inv u32 buffers")
    if len(scores) < tokens * top_k or len(inv) < tokens * top_k:
        raise _lib.InvalidArgument("moe_combine: scores or inv shorter than tokens*top_k")
    _lib.check(_lib.lib().cpq_moe_combine(
        commands.handle, _lib.DTYPES[y.dtype], _ptr(y), len(y), _ptr(scores), _ptr(inv), tokens, top_k, n,
        _ptr(out), len(out)))
