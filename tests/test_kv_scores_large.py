"""Attention for many rows (kernels/kv_attention.hpp) with scores that are capped,
biased or both, where it takes other paths than small calls: workgroups of eight
waves, whose two halves stage tiles in turn (head_dim 128, from 256 query rows for
each compute unit on), and keys that no workgroup shares, so many that the block
ids are fetched again on the way -- with biases from the last keys to the first.

A sample of the rows against float64.  No reference counterpart; semantics in
include/cpq.h.
"""
import numpy as np
import pytest

from cider_press_amd.synthetic import from_bits
from test_kv_scores import ROUNDING, make

KINDS = [dict(cap=30.0), dict(slopes=True), dict(cap=20.0, slopes=True), dict(prefix=True)]


def check_rows(b, bits, rows, window=0):
    """The queries `rows` of the one sequence of `b`, causal; tolerances are those of Scored.check and Scored.expect."""
    (m,), (n,) = b.q_lens, b.kv_lens
    rows = np.asarray(rows)
    pos, j = (n - m + rows)[:, None], np.arange(n)[None, :]
    seen = (j <= pos) | (j < (0 if b.prefix is None else int(b.prefix[0])))
    if window:
        seen &= j > pos - window
    scale, total = b.dim ** -0.5, [0.0, 0.0]
    for h in range(b.heads):
        q, k, v = b.q[rows, h], b.k[0][:, h // b.group], b.v[0][:, h // b.group]
        z = q @ k.T * scale
        if b.cap:
            z = b.cap * np.tanh(z / np.float64(np.float32(b.cap)))
        bias = np.zeros(z.shape) if b.slopes is None else np.float64(b.slopes[h]) * (j - pos)
        z = np.where(seen, z + bias, -np.inf)
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        size = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0).max(1, keepdims=True)
        bias = np.where(seen & (p > 2.0 ** -40), bias, np.nan)
        far = (np.nanmax(bias, 1) - np.nanmin(bias, 1))[:, None]
        off = 2.0 ** -10 * size + 2.0 ** -10 + 2.0 ** -21 * b.cap + 2.0 ** -21 * far
        want, bound = p @ v, off * (p @ np.abs(v))
        got = from_bits(bits[rows, h], b.dtype).astype(np.float64)
        assert np.isfinite(got).all()
        u, err = ROUNDING[b.dtype], np.abs(got - want)
        assert (err <= u * np.abs(want) + (1 + u) * bound + 1e-7).all(), (h, (err - u * np.abs(want) - bound).max())
        total[0] += (err ** 2).sum()
        total[1] += (want ** 2).sum()
    assert total[0] ** 0.5 <= (2.2e-3 if b.dtype == "bf16" else 9e-4) * total[1] ** 0.5 + 1e-7


def sample(rng, m):
    """The first and last queries, those about a tile of 8, and others."""
    return np.unique(np.concatenate([[0, 1, 7, 8, 9, m // 2, m - 9, m - 2, m - 1], rng.integers(0, m, 24)]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gs", [("bf16", 64), ("f16", 32), ("f16", 128)])
@pytest.mark.parametrize("kind", range(len(KINDS)))
@pytest.mark.parametrize("kv_heads,group", [(4, 8), (1, 32)])
def test_eight_waves(device, dtype, gs, kind, kv_heads, group):
    """2100 queries of 32 heads, 262 row tiles of 256: without a mask but the causal one, in a window, over a prefix."""
    rng = np.random.default_rng(kind * 7 + gs + group)
    m, n = 2100, 2611
    what = {**KINDS[kind], "prefix": np.uint32([2400]) if kind > 1 else None}
    b = make(rng, device, (dtype, 128, gs, 16, kv_heads, group), [m], [n], **what, sharp=2.0)
    rows = sample(rng, m)
    check_rows(b, b.run(), rows)
    check_rows(b, b.run(window=700), rows, 700)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,m,n,kv_heads,group", [
    ("bf16", 128, 64, 2049, 5003, 4, 8), ("f16", 128, 64, 2049, 4500, 1, 32),  # eight waves
    ("bf16", 128, 128, 75, 3011, 2, 4), ("f16", 128, 32, 33, 5003, 1, 8), ("bf16", 64, 64, 40, 4477, 2, 3),
    ("f16", 64, 32, 100, 2177, 1, 4), ("bf16", 256, 64, 64, 2500, 1, 2), ("f16", 256, 128, 40, 4200, 1, 4)])
def test_unsplit(device, monkeypatch, dtype, dim, gs, m, n, kv_heads, group):
    """More than 32 tiles for each team that stages them, whose blocks lie in any order; also in a window that ends
    within a later fetch."""
    monkeypatch.setenv("CPQ_SESSION_SCRATCH_MB", "0")  # no room for parts
    rng = np.random.default_rng(m + n + gs)
    for kind in KINDS[:3]:
        b = make(rng, device, (dtype, dim, gs, 16, kv_heads, group), [m], [n], **kind, sharp=2.0)
        rows = sample(rng, m)
        check_rows(b, b.run(), rows)
        check_rows(b, b.run(window=n - m - 300), rows, n - m - 300)
