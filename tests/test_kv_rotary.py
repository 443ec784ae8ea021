"""Position rotation and append in one pass (kernels/kv_cache.hip) against its
definition in float64 and the append's in numpy, bit for bit: a device's
cosines differ from numpy's in the last of 53 bits, which a rounding to T sees
once in 2^40 values.

No reference counterpart for the cache; semantics in include/cpq.h.
"""
import ctypes

import numpy as np
import pytest

from cider_press_amd import _lib
from cider_press_amd.kernels import Buffer
from cider_press_amd.kernels import kv as kkv
from cider_press_amd.synthetic import from_bits, to_bits
from test_kv_cache import GEOMETRIES, NONE, Host, _cache, _rows, quantize

ARRAYS = ("k_q", "k_sb", "v_q", "v_sb")


def rotate(bits, dtype, positions, frequencies, interleaved=False, magnitude=1.0):
    """T patterns [tokens, heads, dim] rotated."""
    x = from_bits(bits, dtype).astype(np.float64)
    half = len(frequencies)
    with np.errstate(all="ignore"):
        angle = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)[None, :]
        c, s = (magnitude * f(angle)[:, None] for f in (np.cos, np.sin))
        first, second = (np.s_[..., 0:2 * half:2], np.s_[..., 1:2 * half:2]) if interleaved else \
            (np.s_[..., :half], np.s_[..., half:2 * half])
        a, b = x[first], x[second]
        y = x.copy()
        y[first], y[second] = a * c - b * s, b * c + a * s
        out = to_bits(y.astype(np.float32), dtype)
    out[..., 2 * half:] = bits[..., 2 * half:]
    return out


def frequencies_of(rotary, base=1e4):
    return (base ** -(np.arange(0, rotary, 2) / rotary)).astype(np.float32)


def _args(**over):
    a = dict(q=4096, qt=512, qh=128, qo=8192, ot=512, oh=128, heads=4, k=4096, kt=256, kh=128, v=4096, vt=256, vh=128,
             slots=4096, positions=4096, tokens=3, frequencies=4096, rotary=128, interleaved=0, magnitude=1.0)
    a.update(over)
    return kkv._pack("kv_append_rotary", kkv._ROTARY_ARGS, *(v or 0 for v in a.values()))


def test_refusals():
    check, c = _lib.lib().cpq_check_kv_append_rotary_args, _cache()
    run = lambda **over: check(ctypes.byref(c), _args(**over))
    assert run() == _lib.OK
    assert run(tokens=0, q=None, k=None, v=None, slots=None, positions=None) == _lib.OK
    assert run(heads=0, q=None, qo=None) == _lib.OK
    assert run(qo=4096) == _lib.OK  # in place
    assert run(oh=3 * 128, ot=128) == _lib.OK
    assert run(rotary=16) == _lib.OK
    assert check(ctypes.byref(c), None) == _lib.INVALID_ARGUMENT
    assert check(None, _args()) == _lib.INVALID_ARGUMENT
    for bad in (dict(rotary=0), dict(rotary=8), dict(rotary=24), dict(rotary=144), dict(rotary=256),
                dict(magnitude=float("nan")), dict(magnitude=float("inf")), dict(heads=65536), dict(q=None),
                dict(qo=None), dict(k=None), dict(v=None), dict(slots=None), dict(positions=None),
                dict(frequencies=None), dict(frequencies=4098), dict(positions=4097), dict(slots=4098), dict(q=4104),
                dict(qo=4104), dict(k=4098), dict(v=4100), dict(qt=513), dict(oh=4), dict(kt=100), dict(vh=1),
                dict(tokens=2**31), dict(tokens=2**28), dict(ot=128), dict(oh=64), dict(qo=4096, ot=1024), dict(kt=2**62)):
        assert run(**bad) == _lib.INVALID_ARGUMENT, bad
    assert _lib.lib().cpq_kv_append_rotary(None, None, None) == _lib.INVALID_ARGUMENT
    # The packed form is the C structure's.
    assert kkv._ROTARY_ARGS.size % 8 == 0 and kkv._SCORES.size % 8 == 0


def test_buffer_checks():
    """The Python layer's checks come before any call of the library."""
    class Cache:
        dtype, n_kv_heads, head_dim, _ref = "bf16", 1, 64, None

    b = lambda n, t: Buffer(None, None, n, t, 4 * n)
    good = dict(q=b(256, "bf16"), k=b(128, "bf16"), v=b(128, "bf16"), slots=b(2, "u32"), positions=b(2, "u32"),
                frequencies=b(32, "f32"), q_out=b(256, "bf16"), tokens=2, n_heads=2)
    for error, over in ((TypeError, dict(positions=b(2, "f32"))), (TypeError, dict(frequencies=b(32, "bf16"))),
                        (TypeError, dict(q=b(256, "f16"))), (_lib.InvalidArgument, dict(slots=b(1, "u32"))),
                        (_lib.InvalidArgument, dict(positions=b(1, "u32"))),
                        (_lib.InvalidArgument, dict(q_out=b(255, "bf16"))),
                        (_lib.InvalidArgument, dict(v=b(127, "bf16"))),
                        (_lib.InvalidArgument, dict(q_strides=(-8, 64)))):
        with pytest.raises(error):
            kkv.kv_append_rotary(None, Cache, **{**good, **over})


class Step:
    """A step's fused rows [tokens, heads + 2 * kv_heads + 1, dim] and its cache, on host and device."""

    def __init__(self, rng, device, dtype, dim, gs, bs, tokens, heads, kv_heads, positions=None):
        self.device, self.dtype, self.dim, self.gs = device, dtype, dim, gs
        self.tokens, self.heads, self.kv_heads = tokens, heads, kv_heads
        self.blocks = -(-tokens // bs) + 2
        self.host = Host(rng, dtype, self.blocks, bs, kv_heads, dim, gs)
        self.rows = np.concatenate([_rows(rng, tokens, n, dim, dtype)[0] for n in (heads + kv_heads, kv_heads, 1)], 1)
        self.slots = rng.permutation(self.blocks * bs)[:tokens].astype(np.uint32)
        self.positions = np.asarray(rng.integers(0, 100000, tokens) if positions is None else positions, np.uint32)

    def upload(self):
        d = self.device
        self.cache = self.host.upload(d)
        self.x = d.upload(self.rows.reshape(-1), self.dtype)
        self.buffers = [d.upload(self.slots, "u32"), d.upload(self.positions, "u32")]
        self.q_out = d.upload(np.full(max(self.tokens * self.heads * self.dim, 8), 0x5A5A, np.uint16), self.dtype)

    def encode(self, cmds, frequencies, **kw):
        h, kvh, d = self.heads, self.kv_heads, self.dim
        strides, n = (self.rows.shape[1] * d, d), len(self.x)
        q_out = kw.pop("q_out", self.q_out)
        kkv.kv_append_rotary(cmds, self.cache, self.x, self.x.slice(h * d, n - h * d),
                             self.x.slice((h + kvh) * d, n - (h + kvh) * d), *self.buffers, frequencies, q_out,
                             self.tokens, h, q_strides=strides, k_strides=strides, v_strides=strides, **kw)

    def want(self, frequencies, **kw):
        """Queries; the host's cache takes keys and values."""
        turned = rotate(self.rows, self.dtype, self.positions, frequencies, **kw)
        h, kvh = self.heads, self.kv_heads
        value = lambda bits: quantize(from_bits(bits, self.dtype).astype(np.float32), self.gs, self.dtype)
        live = self.slots < self.host.n * self.host.bs
        self.host.put(self.slots, value(turned[:, h:h + kvh]), value(self.rows[:, h + kvh:h + 2 * kvh]))
        q = np.full((self.tokens, h, self.dim), 0x5A5A, np.uint16)
        q[live] = turned[live, :h]
        return q

    def check(self, frequencies, **kw):
        self.upload()
        cmds = self.device.commands()
        self.encode(cmds, self.device.upload(frequencies, "f32"), **kw)
        cmds.commit_and_wait()
        self.same(self.want(frequencies, **kw))

    def same(self, q):
        for name, want in zip(ARRAYS, self.host.arrays()):
            assert np.array_equal(getattr(self.cache, name).to_numpy().reshape(want.shape), want), name
        assert np.array_equal(self.q_out.to_numpy()[:q.size].reshape(q.shape), q)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", GEOMETRIES)
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (7, 6, 3), (70, 4, 2)])
def test_append(device, dtype, dim, gs, bs, tokens, heads, kv_heads):
    """Either pairing, all and a part of the dimensions."""
    for i, rotary in enumerate((dim, dim // 2, 16, dim - 16)):
        rng = np.random.default_rng(dim + gs + tokens + i)
        s = Step(rng, device, dtype, dim, gs, bs, tokens, heads, kv_heads)
        s.check(frequencies_of(rotary), interleaved=bool(i & 1) ^ (tokens == 7), magnitude=1.0 if i else 1.25)


@pytest.mark.gpu
def test_many_tokens(device):
    """Several rows to a workgroup."""
    s = Step(np.random.default_rng(3), device, "bf16", 128, 64, 16, 3001, 21, 3)
    s.check(frequencies_of(128, 5e5))
    s = Step(np.random.default_rng(4), device, "f16", 64, 32, 64, 5003, 30, 2)
    s.check(frequencies_of(48), interleaved=True)


@pytest.mark.gpu
def test_many_heads(device):
    """More rows than a grid's second dimension holds."""
    s = Step(np.random.default_rng(2), device, "bf16", 64, 64, 16, 1, 65535, 9)
    s.check(frequencies_of(64))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_and_frequencies(device, interleaved):
    """Positions up to their type's end; angles next to multiples of a quarter turn, of any size; frequencies of 0, below
    0, past 1, and that are not finite."""
    rng = np.random.default_rng(7)
    positions = np.concatenate([[0, 1, 2, 2**24 - 1, 2**24 + 1, 2**31 - 1, 2**31, 2**32 - 1],
                                rng.integers(0, 2**32, 40), rng.integers(0, 2**20, 40)])
    frequencies = frequencies_of(64)
    frequencies[3:15] = [0.0, -0.25, 1.5, 3e3, 1e10, 1e30, 1e-30, np.pi / 2, np.pi / 4, 2 * np.pi, 1e-45, -7.0]
    s = Step(rng, device, "f16", 64, 32, 32, len(positions), 2, 2, positions)
    s.check(frequencies, interleaved=interleaved)
    frequencies[1], frequencies[20] = np.inf, np.nan
    s = Step(rng, device, "bf16", 64, 64, 32, len(positions), 1, 1, positions)
    s.upload()
    cmds = device.commands()
    s.encode(cmds, device.upload(frequencies, "f32"), interleaved=interleaved)
    cmds.commit_and_wait()
    got, want = (from_bits(b, "bf16") for b in (s.q_out.to_numpy()[:len(positions) * 64].reshape(-1, 1, 64),
                                                 s.want(frequencies, interleaved=interleaved)))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    assert np.isnan(from_bits((s.cache.k_sb.to_numpy() >> 16).astype(np.uint16), "bf16")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_special_values(device, dtype):
    """Inf and NaN reach their pair and, in the cache, their group; zeros keep their signs; large values overflow."""
    rng = np.random.default_rng(9)
    s = Step(rng, device, dtype, 128, 32, 16, 9, 1, 1)
    inf, nan, most = (0x7F80, 0x7FC0, 0x7F7F) if dtype == "bf16" else (0x7C00, 0x7E00, 0x7BFF)
    for row in (0, 1, 2):  # query, key, value
        s.rows[0, row, 3], s.rows[1, row, 70], s.rows[2, row, 127] = inf, nan, inf | 0x8000
        s.rows[3, row], s.rows[4, row, ::2] = 0x8000, 0
        s.rows[5, row, :40], s.rows[5, row, 64:90] = most, most
    s.positions[6:] = 0  # not rotated: infinities times a sine of 0
    s.rows[6, :, 5] = inf
    for interleaved in (False, True):
        s.upload()
        cmds = device.commands()
        f = frequencies_of(128)
        s.encode(cmds, device.upload(f, "f32"), interleaved=interleaved)
        outs = [device.alloc_buffer(9 * 128, dtype) for _ in range(2)]
        kkv.kv_gather(cmds, s.cache, s.buffers[0], 9, *outs)
        cmds.commit_and_wait()
        want_q = s.want(f, interleaved=interleaved)
        fresh = s.host.upload(device)
        wants = [device.alloc_buffer(9 * 128, dtype) for _ in range(2)]
        kkv.kv_gather(cmds, fresh, s.buffers[0], 9, *wants)
        cmds.commit_and_wait()
        for got, want in ((s.q_out.to_numpy()[:want_q.size], want_q.reshape(-1)),
                          *((a.to_numpy(), b.to_numpy()) for a, b in zip(outs, wants))):
            g, w = from_bits(got, dtype), from_bits(want, dtype)
            assert np.array_equal(np.isnan(g), np.isnan(w))
            assert np.array_equal(got[~np.isnan(g)], want[~np.isnan(w)])
        assert (~np.isfinite(from_bits(want_q[0], dtype))).sum() == 2 and np.isnan(from_bits(want_q[1], dtype)).sum() == 2


@pytest.mark.gpu
def test_skipped_tokens(device):
    """Padding and slots past the cache: nothing written, the latter reported."""
    s = Step(np.random.default_rng(1), device, "bf16", 128, 64, 16, 40, 3, 2)
    s.slots[[0, 7, 39]] = NONE
    s.check(frequencies_of(128))
    s.slots[5], s.slots[30] = s.blocks * 16, 0xFFFFFFF0
    s.host = Host(np.random.default_rng(2), "bf16", s.blocks, 16, 2, 128, 64)
    s.upload()
    cmds = device.commands()
    f = frequencies_of(128)
    s.encode(cmds, device.upload(f, "f32"))
    with pytest.raises(_lib.InvalidArgument, match="2 slot"):
        cmds.commit_and_wait()
    s.same(s.want(f))
    cmds.commit_and_wait()


@pytest.mark.gpu
def test_layouts(device):
    """In place, heads first, queries left out, nothing at all; broadcast keys."""
    f = frequencies_of(64)
    for interleaved in (False, True):
        s = Step(np.random.default_rng(5), device, "bf16", 64, 64, 16, 37, 5, 1)
        s.upload()
        F, cmds, strides = device.upload(f, "f32"), device.commands(), (8 * 64, 64)
        s.encode(cmds, F, q_out=s.x, q_out_strides=strides, interleaved=interleaved)
        cmds.commit_and_wait()
        want = s.rows.copy()
        want[:, :5] = s.want(f, interleaved=interleaved)
        assert np.array_equal(s.x.to_numpy().reshape(want.shape), want)  # keys and values in their rows stay
        s.upload()
        s.encode(cmds, F, q_out_strides=(64, 37 * 64), interleaved=interleaved)
        cmds.commit_and_wait()
        assert np.array_equal(s.q_out.to_numpy().reshape(5, 37, 64).transpose(1, 0, 2), want[:, :5])
        s.same(s.q_out.to_numpy()[:0].reshape(0))
    none = Host(np.random.default_rng(6), "bf16", 3, 16, 1, 64, 64)
    cache = none.upload(device)
    kkv.kv_append_rotary(cmds, cache, None, s.x.slice(5 * 64, 192), s.x.slice(6 * 64, 64), *s.buffers, F, None, 0, 0)
    cmds.commit_and_wait()
    for name, a in zip(ARRAYS, none.arrays()):
        assert np.array_equal(getattr(cache, name).to_numpy().reshape(a.shape), a)
    s.heads, s.slots = 0, np.arange(37, dtype=np.uint32)
    s.host = Host(np.random.default_rng(6), "bf16", 3, 16, 1, 64, 64)
    s.upload()
    kkv.kv_append_rotary(cmds, s.cache, None, s.x, s.x.slice(64, 64), *s.buffers, F, None, 37, 0, k_strides=(0, 64),
                         v_strides=(0, 64))  # one key and value at 37 positions
    cmds.commit_and_wait()
    s.rows = np.broadcast_to(s.rows[:1], s.rows.shape).copy()
    s.want(f)
    s.same(s.q_out.to_numpy()[:0].reshape(0))


@pytest.mark.gpu
def test_graph(device):
    """A captured call replayed on new inputs, with eager calls in between."""
    s = Step(np.random.default_rng(8), device, "bf16", 128, 64, 16, 30, 4, 2)
    f = frequencies_of(128)
    F = device.upload(f, "f32")
    s.upload()
    cmds = device.commands()
    cmds.begin_capture()
    s.encode(cmds, F)
    graph = cmds.end_capture()
    for i in range(3):
        s.positions = (s.positions + 1000 * i).astype(np.uint32)
        s.buffers[1].write(s.positions)
        s.q_out.write(np.full(len(s.q_out), 0x5A5A, np.uint16))
        graph.launch(cmds)
        cmds.wait()
        s.same(s.want(f))
        s.encode(cmds, F)
        cmds.wait()
        s.same(s.want(f))
