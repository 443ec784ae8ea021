"""Key/value cache: what no query row may see is not seen, whatever it holds --
places never written or left by ended requests, finite or not.

Attention against float64 over the seen keys alone, with bounds that know
nothing of the others (test_kv_cache.py: Batch).
"""
import numpy as np
import pytest

from cider_press_amd import _lib
from test_kv_cache import GEOMETRIES, NAN, Batch

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
