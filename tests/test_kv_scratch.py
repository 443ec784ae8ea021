"""Attention over the key/value cache where the session's scratch is small or
missing: keys are split as far as it goes; and what a call leaves there
(test_kv_cache.py: Batch)."""
import numpy as np
import pytest

from cider_press_amd import _lib
from test_kv_cache import Batch

# Parts of a workgroup of four waves that 1 MiB holds behind the arrival counters.
ROOM = {d: ((1 << 20) - (64 << 10)) // (4 * (d // 8 + 1) * 64 * 16) for d in (64, 128, 256)}


def _session(device, monkeypatch, mib):
    monkeypatch.setenv("CPQ_SESSION_SCRATCH_MB", str(mib))
    cmds = device.commands()
    monkeypatch.delenv("CPQ_SESSION_SCRATCH_MB")
    return cmds


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("short", [1, 2, 3, 4, 9])
def test_room_for_a_few_parts(device, monkeypatch, dim, short):
    """A prompt whose row tiles leave room for `short` parts: its rows, and after it
    on the same session keys that are split."""
    rng = np.random.default_rng(dim + short)
    cmds = _session(device, monkeypatch, 1)
    tiles = max(ROOM[dim] - short - 1, 1)  # of 128 rows, and one a sequence
    q = tiles * 128 // 4 + 3
    b = Batch(rng, device, "bf16", dim, 64, 16, 1, 4, [q], [q + 900])
    first = b.run(cmds=cmds)
    b.check(first)
    assert np.array_equal(b.run(cmds=cmds), first)
    for n in (1, 20):
        after = Batch(rng, device, "bf16", dim, 64, 16, 1, 4, [n], [3000])
        want = after.run(cmds=cmds)
        after.check(want)
        assert np.array_equal(after.run(cmds=cmds), want)


@pytest.mark.gpu
@pytest.mark.parametrize("mib", [0, 1, 2])
@pytest.mark.parametrize("q,kv", [([1], [5000]), ([1, 2, 1], [4000, 2500, 10]), ([70], [1500]), ([1, 60, 3], [3000, 900, 40]),
                                  ([1] * 140, [50] * 139 + [2000])])
def test_small_scratch(device, monkeypatch, mib, q, kv):
    """No scratch, and less than the splits would take; more sequences than one
    workgroup goes over."""
    rng = np.random.default_rng(mib + len(q))
    cmds = _session(device, monkeypatch, mib)
    b = Batch(rng, device, "f16", 128, 64, 16, 2, 4, q, kv)
    first = b.run(cmds=cmds)
    b.check(first)
    assert np.array_equal(b.run(cmds=cmds), first)


@pytest.mark.gpu
def test_query_starts_that_overlap(device):
    """Starts that are not ascending are reported, and leave nothing behind that a
    later call on the session meets."""
    rng = np.random.default_rng(3)
    cmds = device.commands()
    b = Batch(rng, device, "bf16", 64, 64, 16, 1, 4, [640], [2000])
    n = 65
    b.starts = np.array([0, 640] * n, np.uint32)
    b.kv_lens, b.table = b.kv_lens * (2 * n - 1), np.repeat(b.table, 2 * n - 1, 0)
    with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
        b.run(cmds=cmds)
    for q in (1, 20, 70):
        after = Batch(rng, device, "bf16", 64, 64, 16, 1, 4, [q], [3000])
        want = after.run(cmds=cmds)
        after.check(want)
        assert np.array_equal(after.run(cmds=cmds), want)
