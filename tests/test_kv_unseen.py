"""Key/value cache: what no query row may see is not seen, whatever it holds --
places never written or left by ended requests, finite or not.

Attention against float64 over the seen keys alone, with bounds that know
nothing of the others (test_kv_cache.py: Batch).
"""
import numpy as np
import pytest

from cider_press_amd import _lib
from cider_press_amd.synthetic import from_bits, to_bits
from test_kv_cache import GEOMETRIES, NAN, Batch, _prompts, dequantize, quantize

FILLED = GEOMETRIES + [("bf16", 128, 128, 16), ("f16", 64, 64, 16)]
LARGEST = {"bf16": 0x7F7F, "f16": 0x7BFF}  # finite


def _fill(b, what):
    """Puts `what` in every constant that no token wrote: the largest finite scale
    and bias of T (and its negative), or random words."""
    rng, nan, top = np.random.default_rng(99), NAN[b.dtype] * 0x10001, LARGEST[b.dtype]
    for a in (b.host.k_sb, b.host.v_sb):
        free = a == nan
        words = rng.integers(0, 2 ** 32, a.shape, dtype=np.uint32)
        if what == "largest":
            words = np.where(words & 1, top * 0x10001, top * 0x10001 ^ 0x80000000).astype(np.uint32)
        a[free] = words[free]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", FILLED)
@pytest.mark.parametrize("what", ["largest", "random"])
def test_places_past_the_end(device, dtype, dim, gs, bs, what):
    """One token over every length around a tile's end, then several queries of
    several sequences: the last tile holds constants that nobody wrote."""
    rng = np.random.default_rng(dim * gs + len(what))
    kv = [1, 2, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 129, 255, 300]
    b = Batch(rng, device, dtype, dim, gs, bs, 2, 4, [1] * len(kv), kv)
    _fill(b, what)
    b.check(b.run())
    q, kv = [1, 40, 0, 130, 3, 65], [77, 40, 50, 200, 3, 129]
    for causal, window in ((True, 0), (False, 0), (True, 37), (False, 70)):
        b = Batch(rng, device, dtype, dim, gs, bs, 2, 3, q, kv)
        _fill(b, what)
        b.check(b.run(causal, window), causal, window)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 5, 40, 200])
@pytest.mark.parametrize("window", [16, 33, 70, 300])
def test_blocks_behind_the_window(device, q, window):
    """A program that gives blocks back once no query sees them, and clears their
    entries, has no error; the block of the first key that a query sees is one."""
    rng = np.random.default_rng(q + window)
    kv = [q + n for n in (0, 1, 90, 333, 350, 1111)]
    b = Batch(rng, device, "bf16", 128, 64, 16, 2, 4, [q] * len(kv), kv)
    for s, n in enumerate(kv):
        b.table[s, :max(0, n - q + 1 - window) // 16] = 0xFFFFFFFF
    b.check(b.run(window=window), window=window)
    first = max(0, kv[-1] - q + 1 - window) // 16
    b.table[-1, first] = 0xFFFFFFFF
    with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
        b.run(window=window)


BIG = {"bf16": (1e3, 1e8, 1e30, 1.2e38), "f16": (300.0, 2e4, 6e4)}


def _put(b, s, p, k=None, v=None):
    """Token p of sequence s holds keys of size k, values of size v."""
    rng, bs, dim = np.random.default_rng(p), b.host.bs, b.dim
    parts = []
    for size, have in ((k, b.k[s]), (v, b.v[s])):
        x = have[p:p + 1].astype(np.float32) if size is None else \
            (rng.choice([-1.0, 1.0, 0.5, -0.2], (1, b.kv_heads, dim)) * size).astype(np.float32)
        parts.append(quantize(from_bits(to_bits(x, b.dtype), b.dtype).astype(np.float32), b.host.gs, b.dtype))
    slot = np.array([int(b.table[s, p // bs]) * bs + p % bs])
    # (float64 of an unchanged token is not its bits again: only what changes is put.)
    old = [a.copy() for a in b.host.arrays()]
    b.host.put(slot, *parts)
    if k is None:
        b.host.k_q[:], b.host.k_sb[:] = old[0], old[1]
    else:
        b.k[s][p] = dequantize(*parts[0], b.host.gs, b.dtype)
    if v is None:
        b.host.v_q[:], b.host.v_sb[:] = old[2], old[3]
    else:
        b.v[s][p] = dequantize(*parts[1], b.host.gs, b.dtype)


def _rows_close(b, got, rows, causal=True, window=0):
    """As Batch.check, of some rows: bounds of what they see alone."""
    want, bound = b.expect(causal, window)
    out = from_bits(got, b.dtype).astype(np.float64)[rows]
    want, bound = want[rows], bound[rows]
    assert np.isfinite(out).all()
    unit = 2.0 ** -8 if b.dtype == "bf16" else 2.0 ** -11
    err = np.abs(out - want)
    assert (err <= unit * np.abs(want) + bound + 1e-7).all(), (err - bound - unit * np.abs(want)).max()
    assert np.linalg.norm(err) <= (2.2e-3 if b.dtype == "bf16" else 9e-4) * np.linalg.norm(want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", FILLED)
@pytest.mark.parametrize("q", [2, 6, 40, 150])
def test_large_tokens_not_yet_seen(device, dtype, dim, gs, bs, q):
    """Tokens far larger than the others, finite: rows before them are as without."""
    for i, size in enumerate(BIG[dtype]):
        rng = np.random.default_rng(dim + gs + q)
        b = Batch(rng, device, dtype, dim, gs, bs, 1, 3, [q], [q + 75])
        at = [q + 74, q + 74 - q // 2, q + 74 - q // 2 + 1]  # key positions; rows are q + 75 - q ..
        for p in at:
            _put(b, 0, p, None if i % 2 else min(size, 1e4), size)
        _rows_close(b, b.run(), np.arange(q) < q - 1 - q // 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", FILLED)
@pytest.mark.parametrize("q", [1, 5, 40, 150])
def test_large_tokens_behind_the_window(device, dtype, dim, gs, bs, q):
    """The same before every row's window, in the tile where the windows begin and
    in one before it; rows whose window holds them are left out."""
    for size in BIG[dtype]:
        rng = np.random.default_rng(dim + gs + q)
        n, window = q + 200, 45
        b = Batch(rng, device, dtype, dim, gs, bs, 1, 3, [q], [n])
        first = n - q + 1 - window  # of the first row's window
        for p in (3, first - 1, first - 2, first + q // 3):
            _put(b, 0, p, min(size, 1e4), size)
        seen_by = n - q + np.arange(q)  # positions; rows up to q // 3 see the last one
        _rows_close(b, b.run(window=window), seen_by - window + 1 > first + q // 3, window=window) if q > 2 else \
            b.run(window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", FILLED)
@pytest.mark.parametrize("q,n", [(1, 700), (4, 300), (60, 60), (130, 500), (1, 5000)])
def test_large_tokens_without_weight(device, dtype, dim, gs, bs, q, n):
    """Values far larger than the others at keys that no row gives weight to: the
    first token, one in the middle, neighbours.  Later tiles keep their precision,
    and so does the tile itself."""
    for size in BIG[dtype][:3]:
        rng = np.random.default_rng(dim + n)
        b = Batch(rng, device, dtype, dim, gs, bs, 1, 2, [q], [n])
        b.q[:, :, :gs] = 3.0  # the first group of every query
        b.q_bits = to_bits(b.q.astype(np.float32), dtype)
        for p in {0, 1, n // 2 - q // 2}:
            _put(b, 0, p, 1.0, size)
            k = np.zeros((1, 1, dim), np.float32)
            k[..., :gs] = -160.0 / (3.0 * gs) * dim ** 0.5  # a logit of -160
            part = quantize(from_bits(to_bits(k, dtype), dtype).astype(np.float32), gs, dtype)
            vq = quantize(from_bits(to_bits(b.v[0][p:p + 1].astype(np.float32), dtype), dtype).astype(np.float32), gs, dtype)
            b.host.put(np.array([int(b.table[0, p // bs]) * bs + p % bs]), part, vq)
            b.k[0][p], b.v[0][p] = dequantize(*part, gs, dtype), dequantize(*vq, gs, dtype)
        rows = np.arange(q) + n - q > 2  # the first rows of a prompt see little else
        got = b.run()
        want, bound = b.expect()
        unit = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
        err = np.abs(from_bits(got, dtype).astype(np.float64) - want)[rows]
        # bound: 2^-10 of the logits' size, which the three keys raise to 160 for every row.
        limit = unit * np.abs(want[rows]) + bound[rows] / 8 + 1e-7
        assert (err <= limit).all(), (size, (err - limit).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", FILLED)
@pytest.mark.parametrize("q", [1, 4, 70])
def test_every_token_of_another_size(device, dtype, dim, gs, bs, q):
    """Keys' and values' sizes all over the type's range within every tile; each value
    is off by no more than 2^-10 of its own token's largest constant."""
    rng = np.random.default_rng(dim * 3 + q)
    n = 333
    b = Batch(rng, device, dtype, dim, gs, bs, 1, 2, [q], [n])
    low, high = (-20, 20) if dtype == "bf16" else (-8, 12)
    size = np.exp2(rng.uniform(low, high, (n, 1, 1)))
    x = rng.standard_normal((n, 1, dim)).clip(-4, 4) * size
    kx = rng.standard_normal((n, 1, dim)) * np.exp2(rng.uniform(-9, 0, (n, 1, 1)))
    parts = [quantize(from_bits(to_bits(a.astype(np.float32), dtype), dtype).astype(np.float32), gs, dtype) for a in (kx, x)]
    j = np.arange(n)
    b.host.put(b.table[0][j // bs] * bs + j % bs, *parts)
    b.k[0], b.v[0] = (dequantize(*p, gs, dtype) for p in parts)
    want, bound = b.expect()
    # What bound does not have: 2^-10 of a token's largest value, by its weight.
    top = b.v[0].copy()
    b.v[0] = np.broadcast_to(np.abs(top).max(-1, keepdims=True) * 1.2, top.shape)
    own, _ = b.expect()
    b.v[0] = top
    got = from_bits(b.run(), dtype).astype(np.float64)
    unit = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    tiny = 2.0 ** -24 if dtype == "f16" else 0.0
    err = np.abs(got - want)
    assert (err <= unit * np.abs(want) + bound + 2.0 ** -10 * own + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gs", [("bf16", 64), ("f16", 32)])
def test_large_tokens_of_many_prompts(device, dtype, gs):
    """Enough row tiles for workgroups of eight waves: the newest token of every
    prompt is far larger than the others, and what no token wrote as large."""
    b = _prompts(np.random.default_rng(gs + 5), device, dtype, gs)
    last = b.starts[1:] - 1
    for i, n in enumerate(b.kv_lens):
        _put(b, i, n - 1, 100.0, BIG[dtype][-1 - i % 2])
    _fill(b, "largest")
    rows = np.ones(b.tokens, bool)
    rows[last] = False
    got = b.run()
    _rows_close(b, got, rows)
    assert np.array_equal(b.run(), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", FILLED)
@pytest.mark.parametrize("q", [3, 50])
def test_not_finite_beside_large(device, dtype, dim, gs, bs, q):
    """Rows whose queries are Inf or NaN, a token of NaN and one far larger than the
    others behind the rows looked at: those stay as they are."""
    rng = np.random.default_rng(dim + q)
    n = q + 80
    b = Batch(rng, device, dtype, dim, gs, bs, 1, 3, [q], [n])
    _put(b, 0, n - 1, 50.0, BIG[dtype][-1])
    slot = int(b.table[0, (n - 2) // bs]) * bs + (n - 2) % bs
    b.host.v_sb[slot // bs, :, slot % bs // 4, :, slot % 4] = NAN[dtype] * 0x10001
    b.host.k_sb[slot // bs, :, slot % bs] = NAN[dtype] * 0x10001
    inf = 0x7F80 if dtype == "bf16" else 0x7C00
    b.q_bits[0, 0, 5], b.q_bits[0, 1, dim - 1] = inf, NAN[dtype]
    got = b.run()
    rows = np.arange(q) < q - 2
    rows[0] = False
    if rows.any():
        _rows_close(b, got, rows)
    # Of the first row's heads the third's query is finite.
    want, bound = b.expect()
    first = from_bits(got, dtype).astype(np.float64)[0]
    unit = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    assert not np.isfinite(first[:2]).any()
    assert (np.abs(first[2] - want[0, 2]) <= unit * np.abs(want[0, 2]) + bound[0, 2] + 1e-7).all()
    assert np.isnan(from_bits(got[-2:], dtype)).all()
