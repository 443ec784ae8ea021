"""Attention over the 4-bit key/value cache with capped scores, biases that
depend on distance, and prefixes (kernels/kv_attention.hpp, kernels/kv_decode.hpp)
against float64.

No reference counterpart; semantics in include/cpq.h.
"""
import ctypes

import numpy as np
import pytest

from cider_press_amd import _lib
from cider_press_amd.kernels import Buffer
from cider_press_amd.kernels import kv as kkv
from cider_press_amd.synthetic import from_bits, to_bits
from test_kv_cache import GEOMETRIES, Batch, _attention, _cache, _close, _rows


def _scores(softcap=0.0, slopes=0, prefix=0):
    return kkv._pack("op", kkv._SCORES, softcap, slopes, prefix)


def test_refusals():
    check, c = _lib.lib().cpq_check_kv_attention_scored_args, _cache()
    run = lambda scores, **over: check(ctypes.byref(c), _attention(**over), scores)
    for good in (_scores(), _scores(30.0), _scores(1024.0), _scores(1e-40), _scores(0.0, 4096, 4096)):
        assert run(good) == _lib.OK
        assert run(good, tokens=0, q=None, out=None) == _lib.OK
    assert run(None) == _lib.INVALID_ARGUMENT
    for bad in (_scores(-1.0), _scores(float("nan")), _scores(float("inf")), _scores(1024.5), _scores(30.0, 4098),
                _scores(30.0, 0, 4097)):
        assert run(bad) == _lib.INVALID_ARGUMENT
    for bad in (dict(heads=3), dict(q=4098), dict(out=None), dict(scale=0.0), dict(ot=128), dict(lens=None)):
        assert run(_scores(30.0), **bad) == _lib.INVALID_ARGUMENT, bad
    assert check(None, _attention(), _scores()) == _lib.INVALID_ARGUMENT
    assert check(ctypes.byref(c), None, _scores()) == _lib.INVALID_ARGUMENT
    assert _lib.lib().cpq_kv_attention_scored(None, None, None, None) == _lib.INVALID_ARGUMENT


def test_buffer_checks():
    class Cache:
        dtype, n_kv_heads, head_dim, _ref = "bf16", 1, 64, None

    def b(n, t):
        buf = Buffer(None, 4096, n, t, 4 * n)
        buf._owner = buf  # no memory of its own
        return buf

    good = dict(q=b(256, "bf16"), block_table=b(4, "u32"), max_blocks=2, query_starts=b(3, "u32"), kv_lens=b(2, "u32"),
                out=b(256, "bf16"), tokens=2, n_heads=2, n_seqs=2, max_q=1, max_kv=5, scale=0.1)
    for error, over in ((TypeError, dict(slopes=b(2, "bf16"))), (_lib.InvalidArgument, dict(slopes=b(1, "f32"))),
                        (TypeError, dict(prefix_lens=b(2, "f32"))),
                        (_lib.InvalidArgument, dict(prefix_lens=b(1, "u32"))),
                        (_lib.InvalidArgument, dict(kv_lens=b(1, "u32"))), (_lib.InvalidArgument, dict(window=-1))):
        with pytest.raises(error):
            kkv.kv_attention_scored(None, Cache, **{**good, **over})


def standard_slopes(heads):
    return (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32)


# What a value is off by, relative, when rounded to 8 or 11 bits: half a unit of the last one.
ROUNDING = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Scored(Batch):
    """cap, slopes ([heads] or None), prefix ([sequences] or None) on top of a Batch."""

    cap, slopes, prefix = 0.0, None, None

    def encode(self, cmds, causal=True, window=0, max_q=None, max_kv=None, scale=None):
        n = self.tokens
        kkv.kv_attention_scored(cmds, *self.keep[:3], self.width, *self.keep[3:6], n, self.heads, len(self.kv_lens),
                                max(self.q_lens) if max_q is None else max_q,
                                max(self.kv_lens) if max_kv is None else max_kv, scale or self.dim ** -0.5,
                                causal=causal, window=window, softcap=self.cap, slopes=self.keep[6],
                                prefix_lens=self.keep[7], out_strides=None)

    def run(self, causal=True, window=0, cmds=None, cache=None, **kw):
        d = self.device
        up = lambda a, t="u32": None if a is None else d.upload(np.asarray(a, np.uint32 if t == "u32" else np.float32)
                                                                 .reshape(-1), t)
        out = d.upload(np.full(self.tokens * self.heads * self.dim, 0x5A5A, np.uint16), self.dtype)
        cmds = cmds or d.commands()
        self.keep = (cache or self.host.upload(d), d.upload(self.q_bits.reshape(-1), self.dtype), up(self.table),
                     up(self.starts), up(self.kv_lens), out, up(self.slopes, "f32"), up(self.prefix))
        self.encode(cmds, causal, window, **kw)
        cmds.commit_and_wait()
        return out.to_numpy().reshape(self.tokens, self.heads, self.dim)

    def check(self, bits, causal=True, window=0, scale=None):
        """The result is rounded once, from what `bound` says."""
        want, bound = self.expect(causal, window, scale)
        got = from_bits(bits, self.dtype).astype(np.float64)
        assert np.isfinite(got).all()
        u, err = ROUNDING[self.dtype], np.abs(got - want)
        assert (err <= u * np.abs(want) + (1 + u) * bound + 1e-7).all(), (err - u * np.abs(want) - bound).max()
        # A rounding's root mean square is 0.58 of half a step, over a power of two 0.0015 of the values' in bf16 and
        # 0.0002 in f16; the operands' (2^-12 each) add to that.
        assert np.linalg.norm(err) <= (2.2e-3 if self.dtype == "bf16" else 9e-4) * np.linalg.norm(want) + 1e-7

    def expect(self, causal=True, window=0, scale=None):
        """As Batch's.  A cap's slope is at most 1, so what a score is off by stays that at most; the cap adds 2^-22 of
        itself, a bias 2^-23 of the largest that a weight above 2^-40 has (one rounding each of product and sum)."""
        scale = scale or self.dim ** -0.5
        out, bound = np.zeros(self.q.shape), np.zeros(self.q.shape)
        for i, (m, n) in enumerate(zip(self.q_lens, self.kv_lens)):
            pos, j = np.arange(n - m, n)[:, None], np.arange(n)[None, :]
            seen = np.ones((m, n), bool)
            if causal:
                seen &= (j <= pos) | (j < (0 if self.prefix is None else int(self.prefix[i])))
            if window:
                seen &= j > pos - window
            at = slice(self.starts[i], self.starts[i + 1])
            for h in range(self.heads if m and n else 0):
                q, k, v = self.q[at, h], self.k[i][:, h // self.group], self.v[i][:, h // self.group]
                z = q @ k.T * scale
                if self.cap:
                    z = self.cap * np.tanh(z / np.float64(np.float32(self.cap)))
                bias = 0.0 if self.slopes is None else np.float64(self.slopes[h]) * (j - pos)
                z = np.where(seen, z + bias, -np.inf)
                top = z.max(1, keepdims=True)
                p = np.exp(z - np.where(np.isfinite(top), top, 0))
                total = p.sum(1, keepdims=True)
                p /= np.where(total == 0, 1, total)
                size = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0).max(1, keepdims=True)
                bias = np.where(seen & (p > 2.0 ** -40), bias, np.nan)
                with np.errstate(all="ignore"):
                    far = np.nan_to_num(np.fmax.reduce(bias, 1) - np.fmin.reduce(bias, 1))[:, None]
                off = 2.0 ** -10 * size + 2.0 ** -10 + 2.0 ** -21 * self.cap + 2.0 ** -21 * far
                out[at, h] = p @ v
                bound[at, h] = off * (p @ np.abs(v))
        return out, bound


def make(rng, device, shape, q, kv, cap=0.0, slopes=None, prefix=None, sharp=1.0):
    """shape: dtype, dim, gs, bs, kv_heads, group."""
    b = Scored(rng, device, *shape, q, kv, sharp=sharp)
    b.cap, b.prefix = cap, prefix
    b.slopes = standard_slopes(b.heads) if slopes is True else slopes
    return b


KINDS = [dict(cap=3.0), dict(slopes=True), dict(prefix=True), dict(cap=50.0, slopes=True, prefix=True)]


def _kind(rng, kind, kv):
    return {**kind, "prefix": rng.integers(0, np.asarray(kv) + 1) if kind.get("prefix") else None}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", GEOMETRIES)
@pytest.mark.parametrize("kind", range(4))
def test_one_token(device, dtype, dim, gs, bs, kind):
    rng = np.random.default_rng(dim * gs + kind)
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 300]
    b = make(rng, device, (dtype, dim, gs, bs, 2, [1, 4, 7, 3][kind]), [1] * len(kv), kv, **_kind(rng, KINDS[kind], kv),
             sharp=3.0)
    b.check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", GEOMETRIES)
@pytest.mark.parametrize("kind", range(4))
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 37), (False, 0), (False, 70)])
def test_queries(device, dtype, dim, gs, bs, kind, causal, window):
    """Many queries of several sequences, with cached keys before them or none; and few."""
    rng = np.random.default_rng(dim + gs + kind)
    for q, kv in (([1, 40, 0, 130, 3, 65], [77, 40, 50, 200, 3, 129]), ([1, 5, 0, 3], [77, 5, 50, 200])):
        b = make(rng, device, (dtype, dim, gs, bs, 2, [1, 4, 3, 2][kind]), q, kv, **_kind(rng, KINDS[kind], kv), sharp=2.0)
        b.check(b.run(causal, window), causal, window)


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-40, 1e-6, 0.5, 1.0, 30.0, 1000.0, 1024.0])
@pytest.mark.parametrize("sharp", [1e-3, 1.0, 300.0])
def test_caps(device, cap, sharp):
    """Scores far below a cap, about it and far past it, at few and many queries."""
    for q in ([1, 3], [1, 70]):
        b = make(np.random.default_rng(int(sharp)), device, ("bf16", 64, 32, 16, 1, 4), q, [90, 200], cap=cap, sharp=sharp)
        b.check(b.run())
        b = make(np.random.default_rng(int(sharp)), device, ("f16", 128, 64, 16, 1, 2), q, [90, 200], cap=cap, sharp=sharp)
        b.check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 60])
def test_slopes(device, q):
    """Slopes of 0, below 0, large; without a mask, where the keys of a negative bias and of a positive one are far; the
    largest, which leave one key; NaN, which is its own head's."""
    rng = np.random.default_rng(q)
    for dtype, gs in (("bf16", 64), ("f16", 32)):
        slopes = np.float32([0.0, -0.5, 3.0, 1e4, -1e4, 1e-6, 2.0 ** -8, -2.0])
        for causal in (True, False):
            b = make(rng, device, (dtype, 64, gs, 16, 2, 4), [q, q], [700, 133], slopes=slopes)
            b.check(b.run(causal), causal)
        b.slopes = np.float32([1e38, -1e38, np.inf, -np.inf, 3e38, 2.0 ** 96, -2.0 ** 97, 0.0])
        got = b.run()
        b.slopes = np.clip(b.slopes, np.float32(-2.0 ** 96), np.float32(2.0 ** 96))
        b.check(got)
        b.slopes = np.float32([0.5, np.nan, 0.25, 0.0, 1.0, 2.0, np.nan, 0.1])
        got = from_bits(b.run(), dtype)
        assert np.isnan(got[:, [1, 6]]).all() and np.isfinite(np.delete(got, [1, 6], 1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 2, 40, 200])
def test_prefixes(device, q):
    """Prefixes of nothing, inside a tile and a block, at their ends, of all, past the end; more queries than keys, whose
    first stand before key 0 and see the prefix only; a window before it; none where nothing is masked."""
    rng = np.random.default_rng(q)
    kv = [300] * 7 + [q // 2, q]
    prefix = [0, 1, 31, 64, 299, 300, 2 ** 32 - 1, 3, 2]
    for dtype in ("bf16", "f16"):
        b = make(rng, device, (dtype, 128, 64, 16, 1, 3), [q] * 9, kv, prefix=np.uint32(prefix))
        out = b.run()
        b.check(out)
        b.check(b.run(window=45), window=45)
        b.check(b.run(causal=False), causal=False)
        b.prefix = np.zeros(9, np.uint32)
        plain = b.run()
        b.check(plain)
        b.prefix = None
        b.cap = 0.0
        want = b.run()  # nothing of the three
        b.check(want)
        assert np.array_equal(Batch.run(b), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,group,q,n", [("bf16", 64, 32, 7, 1, 9000), ("f16", 64, 64, 1, 3, 4200),
                                                     ("bf16", 128, 128, 4, 1, 16500), ("f16", 128, 32, 2, 90, 5000),
                                                     ("bf16", 256, 64, 2, 1, 3000), ("bf16", 64, 64, 4, 100, 7000),
                                                     ("bf16", 256, 64, 2, 64, 2500)])
def test_one_long_sequence(device, dtype, dim, gs, group, q, n):
    """Keys split over workgroups and joined."""
    rng = np.random.default_rng(n)
    for kind in (dict(cap=20.0), dict(slopes=True), dict(slopes=True, cap=5.0, prefix=np.uint32([n - q // 2]))):
        b = make(rng, device, (dtype, dim, gs, 16, 1, group), [q], [n], **kind, sharp=2.0)
        b.check(b.run())
    b.check(b.run(window=4500), window=4500)


@pytest.mark.gpu
def test_many_sequences(device):
    """A mixture of prompts, single tokens and requests without any; and more sequences than one pass of the search."""
    rng = np.random.default_rng(12)
    q = [1, 300, 1, 0, 77, 1, 1, 129, 20]
    kv = [500, 300, 1, 40, 900, 1300, 64, 2000, 21]
    for kind in (dict(cap=30.0, slopes=True, prefix=rng.integers(0, np.asarray(kv) + 1)), dict(slopes=True)):
        for dtype, gs in (("bf16", 64), ("f16", 32)):
            b = make(rng, device, (dtype, 128, gs, 16, 2, 7), q, kv, **kind, sharp=1.5)
            b.check(b.run())
    kv = rng.integers(1, 90, 300)
    b = make(rng, device, ("bf16", 64, 64, 16, 1, 2), [1] * 300, kv, cap=4.0, slopes=True,
             prefix=rng.integers(0, kv + 1), sharp=3.0)
    b.check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 40])
def test_masked_and_poisoned(device, q):
    """Inf and NaN in keys and values that no row sees: future tokens behind the prefix, tokens before a window, what a
    block holds past the sequence's end.  A seen one reaches the rows that see it."""
    rng = np.random.default_rng(q)
    kinds = (dict(cap=5.0), dict(slopes=True, cap=5.0), dict(slopes=True))
    for kind in kinds:
        b = make(rng, device, ("bf16", 128, 64, 16, 2, 4), [q, q], [100, 57], **kind)
        for i, n in enumerate(b.kv_lens):
            for p in range(0, n - q - 19):
                slot = b.table[i, p // 16] * 16 + p % 16
                b.host.k_sb[slot // 16, :, slot % 16] = 0x7F80FF80
                b.host.v_sb[slot // 16, :, slot % 16 // 4, :, slot % 4] = 0x7FC07F80
        b.check(b.run(window=20), window=20)
        c = make(rng, device, ("bf16", 128, 64, 16, 2, 4), [q + 3], [90], **kind, prefix=np.uint32([20]))
        clean = c.run()
        slot = int(c.table[0, 89 // 16]) * 16 + 89 % 16
        c.host.k_sb[slot // 16, :, slot % 16] = 0x7FC07FC0
        c.host.v_sb[slot // 16, :, slot % 16 // 4, :, slot % 4] = 0x7FC07FC0
        got = c.run()
        assert _close(got[:-1], clean[:-1], "bf16")
        assert np.isnan(from_bits(got[-1], "bf16")).all()
        c.prefix[0] = 90  # all see it
        assert np.isnan(from_bits(c.run(), "bf16")).all()


@pytest.mark.gpu
def test_key_sizes_apart(device):
    """Tokens of very different sizes, taken in passes: each score capped and biased once."""
    rng = np.random.default_rng(3)
    for q in (1, 50):
        for dtype in ("bf16", "f16"):
            b = make(rng, device, (dtype, 64, 32, 16, 1, 4), [q], [150], cap=10.0, slopes=True)
            far = [3, 40, 41, 77, 149]
            for p in far:
                slot = int(b.table[0, p // 16]) * 16 + p % 16
                for arr, x in ((b.host.k_sb, b.k), (b.host.v_sb, b.v)):
                    at = (slot // 16, slice(None), slot % 16) if arr is b.host.k_sb else \
                        (slot // 16, slice(None), slot % 16 // 4, slice(None), slot % 4)
                    sb = arr[at]
                    s, o = (from_bits((sb >> sh & 0xFFFF).astype(np.uint16), dtype) for sh in (0, 16))
                    size = 2.0 ** 8 if dtype == "bf16" else 2.0 ** 5
                    arr[at] = to_bits(s * size, dtype).astype(np.uint32) | to_bits(o * size, dtype).astype(np.uint32) << 16
                    x[0][p] *= size
            b.check(b.run())


@pytest.mark.gpu
def test_graph_and_reports(device):
    """A captured call replayed with eager ones in between; what the device finds wrong is reported."""
    rng = np.random.default_rng(1)
    for q, kv in (([1, 1, 1], [40, 700, 5]), ([30, 1, 90], [40, 700, 90])):
        b = make(rng, device, ("f16", 128, 64, 16, 2, 3), q, kv, cap=8.0, slopes=True, prefix=np.uint32([3, 0, 60]))
        cmds = device.commands()
        want = b.run(cmds=cmds)
        b.check(want)
        out = b.keep[5]
        cmds.begin_capture()
        b.encode(cmds)
        graph = cmds.end_capture()
        for _ in range(3):
            out.write(np.zeros(len(out), np.uint16))
            graph.launch(cmds)
            cmds.wait()
            assert np.array_equal(out.to_numpy().reshape(want.shape), want)
            b.encode(cmds)
            cmds.wait()
            assert np.array_equal(out.to_numpy().reshape(want.shape), want)
    with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
        b.run(max_q=40)
    b.table[2, 0] = 0x7FFFFFFF
    with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
        b.run()


@pytest.mark.gpu
def test_little_scratch(device, monkeypatch):
    """Sessions whose scratch has no room for parts."""
    rng = np.random.default_rng(2)
    for q, n in ((1, 3000), (64, 1500)):
        b = make(rng, device, ("bf16", 128, 64, 16, 1, 4), [q], [n], cap=10.0, slopes=True)
        for mb in ("0", "1"):
            monkeypatch.setenv("CPQ_SESSION_SCRATCH_MB", mb)
            b.check(b.run())
        monkeypatch.delenv("CPQ_SESSION_SCRATCH_MB")


@pytest.mark.gpu
def test_distances_past_24_bits(device):
    """Keys so far apart that their distance is no 32-bit float: the anchor's side counts.  (One block of 1024 tokens named
    by every entry of a long table.)"""
    rng = np.random.default_rng(5)
    dim, gs, bs, entries = 64, 64, 1024, 17000
    n = entries * bs - 7
    b = make(rng, device, ("bf16", dim, gs, bs, 1, 2), [1], [bs], slopes=np.float32([0.01, 1.0]))
    k, v = b.k[0], b.v[0]
    # With a slope of 0.01 the keys 30000 back have e^-300 of a weight: the last 30 blocks are all.
    b.width, tail = entries, 30
    b.table = np.full((1, entries), b.table[0, 0], np.uint32)
    b.kv_lens = [n]
    got = from_bits(b.run(), "bf16").astype(np.float64)
    b.kv_lens, b.q_lens = [tail * bs - 7], [1]
    b.k, b.v = [np.tile(k, (tail, 1, 1))[:-7]], [np.tile(v, (tail, 1, 1))[:-7]]
    want, bound = b.expect()
    assert (np.abs(got - want) <= ROUNDING["bf16"] * np.abs(want) + bound + 1e-7).all()
