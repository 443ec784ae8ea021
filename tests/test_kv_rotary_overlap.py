"""kv_append_rotary refuses a place for the rotated queries that shares bytes with
what the call reads (csrc/kv.cpp), and takes slices of one fused buffer that do not.

No reference counterpart; semantics in include/cpq.h.
"""
import ctypes
import itertools
import random

import pytest

from cider_press_amd import _lib
from cider_press_amd.kernels import kv as kkv
from test_kv_cache import _cache

BASE, D = 1 << 24, 64
FAR = 1 << 28  # apart from all else


def verdict(tokens, heads, q, q_out, k, v, slots=FAR, positions=FAR, frequencies=FAR, kv_heads=1):
    """None, or what q_out overlaps.  q, q_out, k, v: (byte address, token stride, head stride)."""
    args = kkv._pack("op", kkv._ROTARY_ARGS, *q, *q_out, heads, *k, *v, slots, positions, tokens, frequencies, D, 0, 1.0)
    st = _lib.lib().cpq_check_kv_append_rotary_args(ctypes.byref(_cache(dim=D, heads=kv_heads)), args)
    if st == _lib.OK:
        return None
    assert st == _lib.INVALID_ARGUMENT
    message = _lib.last_error()
    assert "q_out overlaps " in message, message
    return message.rsplit(" ", 1)[1]


def at(elements):
    return BASE + 2 * elements


def test_one_fused_row():
    """[5 queries | 2 keys | 2 values | a spare head] a token."""
    row, far = 10 * D, (FAR * 2, 5 * D, D)
    q, k, v = (at(0), row, D), (at(5 * D), row, D), (at(7 * D), row, D)
    go = lambda q_out, tokens=7, heads=5, **kw: verdict(tokens, heads, kw.pop("q", q), q_out, k, v, kv_heads=2, **kw)
    assert go(far) is None
    assert go(q) is None  # in place
    assert go((at(D), row, D)) == "q"  # a head further: keys too, but the queries are looked at first
    assert go((at(4 * D), row, D), q=far) == "k"
    assert go((at(6 * D), row, D), q=far) == "k"
    assert go((at(8 * D), row, D), q=far) == "v"
    assert go((at(5 * D), row, D), heads=1, q=far) == "k"
    assert go((at(9 * D), row, D), heads=1) is None  # the spare
    assert go((at(9 * D), row, D), heads=2, q=far) is None  # and the next token's first query's, which is nobody's here
    assert go((at(9 * D), row, D), heads=2) == "q"
    assert go((at(9 * D), row, D), heads=2, tokens=1) is None  # there is no next
    assert go((at(10 * D), 4 * D, D), heads=4, q=far) == "k"  # other rows among them
    assert go((at(70 * D), 4 * D, D), heads=4) is None  # behind them
    assert go((at(8), row, D), heads=1) == "q"
    assert go((at(9 * D + 8), row, D), heads=1) == "q"  # the next token's by 8
    for name in ("slots", "positions", "frequencies"):
        assert go((at(100 * D), 5 * D, D), **{name: at(100 * D + 6)}) == name
        assert go((at(100 * D), 5 * D, D), **{name: at(135 * D)}) is None
        assert go((at(100 * D), 5 * D, D), **{name: at(135 * D) - 4}) == name
        assert go((at(9 * D), row, D), heads=1, **{name: at(30 * D)}) is None  # in a gap of q_out's rows


def test_heads_side_by_side():
    """[heads][query | key | value] a token, and a key and a value a head behind the queries."""
    row, head = 12 * D, 3 * D
    q, k, v = (at(0), row, head), (at(D), row, head), (at(2 * D), row, head)
    far = (FAR * 2, 4 * D, D)
    assert verdict(6, 4, q, q, k, v, kv_heads=4) is None
    assert verdict(6, 4, far, q, k, v, kv_heads=4) is None
    assert verdict(6, 4, far, k, (FAR, row, head), v, kv_heads=4) is None
    assert verdict(6, 4, far, k, q, k, kv_heads=4) == "v"
    assert verdict(6, 4, far, (at(8), row, head), k, v, kv_heads=4) == "k"
    row, pair = 9 * D, 2 * D
    k, v = (at(5 * D), row, pair), (at(6 * D), row, pair)
    assert verdict(6, 5, far, (at(0), row, D), k, v, kv_heads=2) is None  # heads at other distances
    assert verdict(6, 6, far, (at(0), row, D), k, v, kv_heads=2) == "k"
    assert verdict(1, 300, far, (at(0), 0, D), (at(2 * D), 0, 299 * D), v, kv_heads=300) == "k"  # pairs not gone through


@pytest.mark.parametrize("seed", range(4))
def test_every_layout(seed):
    """Against the bytes themselves, at small strides."""
    rng, seen = random.Random(seed), {True: 0, False: 0}
    for _ in range(4000):
        tokens, heads, kv_heads = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 3)
        token = 8 * rng.randint(0, 70)
        strides = lambda: (token, 8 * rng.choice([8, 8, 9, 16, 24, rng.randint(0, 40)]))
        place = lambda: (BASE + 16 * rng.randint(0, 400), *strides())
        q_out, k, v = place(), place(), (FAR, token, D)
        spread = lambda x, n: {x[0] // 2 + t * x[1] + h * x[2] + i for t, h, i in
                               itertools.product(range(tokens), range(n), range(0, D, 8))}
        out = spread(q_out, heads)
        if len(out) < tokens * heads * D // 8 or not rows_apart(tokens, heads, *q_out[1:]):
            continue
        want = bool(out & spread(k, kv_heads))
        assert (verdict(tokens, heads, (FAR * 2, 8 * D, D), q_out, k, v, kv_heads=kv_heads) == "k") == want
        seen[want] += 1
    assert min(seen.values()) > 150


def rows_apart(tokens, heads, t, h):
    """Whether the call takes these strides for an output at all."""
    return ((heads == 1 or h >= D) and (tokens == 1 or t >= (heads - 1) * h + D)) or \
        ((tokens == 1 or t >= D) and (heads == 1 or h >= (tokens - 1) * t + D))
