"""Key/value cache in 4 bits (kernels/kv_cache.hip, kernels/kv_attention.hip):
release and plan against a model on Python lists, append and gather against
the format's definition in numpy (bit for bit), attention against float64.

No reference counterpart (its KV cache holds dense T), so these are the
semantics stated in include/cpq.h.
"""
import ctypes

import numpy as np
import pytest

from cider_press_amd import _lib
from cider_press_amd.kernels import Buffer
from cider_press_amd.kernels import kv as kkv
from cider_press_amd.synthetic import from_bits, to_bits

NONE = kkv.NO_SLOT
NAN = {"bf16": 0x7FC0, "f16": 0x7E00}


# ---------------------------------------------------------------------------
# Refusals (no GPU)
# ---------------------------------------------------------------------------

def _cache(**over):
    c = dict(dtype="bf16", dim=128, heads=2, gs=64, block=16, n=8, ptr=4096)
    c.update(over)
    q = c["n"] * c["heads"] * c["block"] * (c["dim"] // 8)
    sb = c["n"] * c["heads"] * c["block"] * (c["dim"] // max(c["gs"], 1))
    a = kkv._CacheArgs(_lib.DTYPES[c["dtype"]], c["dim"], c["heads"], c["gs"], c["block"], c["n"],
                       c["ptr"], c.get("k_q_len", q), c["ptr"], c.get("k_sb_len", sb), c["ptr"], c.get("v_q_len", q),
                       c.get("v_sb", c["ptr"]), c.get("v_sb_len", sb))
    return a


def test_cache_refusals():
    check = _lib.lib().cpq_check_kv_cache
    assert check(ctypes.byref(_cache())) == _lib.OK
    assert check(ctypes.byref(_cache(n=0))) == _lib.OK
    assert check(None) == _lib.INVALID_ARGUMENT
    for bad in (dict(dtype="f32"), dict(dtype="u32"), dict(block=8), dict(block=24), dict(block=2048), dict(heads=0),
                dict(gs=0), dict(gs=48), dict(dim=0), dict(k_q_len=1), dict(k_sb_len=1), dict(v_q_len=1),
                dict(v_sb_len=1), dict(ptr=None), dict(ptr=4100), dict(v_sb=None), dict(n=2**28),
                dict(n=2**61, k_q_len=0)):
        assert check(ctypes.byref(_cache(**bad))) == _lib.INVALID_ARGUMENT, bad
    for missing in (dict(dim=96, gs=32), dict(dim=192), dict(gs=16), dict(dim=512, gs=64), dict(dim=256, gs=256)):
        assert check(ctypes.byref(_cache(**missing))) == _lib.KERNEL_NOT_FOUND, missing
        assert "head_dim" in _lib.last_error()


def test_cache_words():
    for dim, gs in ((64, 32), (64, 64), (128, 32), (128, 128), (256, 128)):
        q, sb = ctypes.c_size_t(), ctypes.c_size_t()
        a = _cache(dim=dim, gs=gs, ptr=None)
        assert _lib.lib().cpq_kv_cache_words(ctypes.byref(a), ctypes.byref(q), ctypes.byref(sb)) == _lib.OK
        assert (q.value, sb.value) == (8 * 2 * 16 * dim // 8, 8 * 2 * 16 * dim // gs)


def _attention(**over):
    a = dict(q=4096, qt=512, qh=128, out=8192, ot=512, oh=128, tokens=3, heads=4, table=4096, max_blocks=4,
             starts=4096, lens=4096, seqs=2, max_q=2, max_kv=10, scale=0.1, causal=1, window=0)
    a.update(over)
    return kkv._attention_args(*(v or 0 for v in a.values()))


def test_attention_refusals():
    check, c = _lib.lib().cpq_check_kv_attention_args, _cache()
    run = lambda **over: check(ctypes.byref(c), _attention(**over))
    assert run() == _lib.OK
    assert run(tokens=0, q=None, out=None) == _lib.OK
    assert run(seqs=0, table=None) == _lib.OK
    assert run(qt=0, qh=0) == _lib.OK  # broadcast queries
    assert run(oh=3 * 128, ot=128) == _lib.OK  # heads first
    assert check(ctypes.byref(c), None) == _lib.INVALID_ARGUMENT
    for bad in (dict(heads=0), dict(heads=3), dict(heads=2**17), dict(qt=513), dict(qh=4), dict(ot=100), dict(q=None),
                dict(out=None), dict(q=4098), dict(out=4104), dict(table=None), dict(starts=None), dict(lens=None),
                dict(lens=4098), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(seqs=2**17), dict(max_blocks=2**31), dict(tokens=2**31),
                dict(oh=64), dict(ot=128), dict(oh=128, ot=128), dict(oh=256, ot=128), dict(qt=2**62)):
        assert run(**bad) == _lib.INVALID_ARGUMENT, bad


def test_ops_refuse_without_session():
    L = _lib.lib()
    assert L.cpq_kv_release(None, *[None] * 3, 0, 0, 16, None, 0, None, None, None) == _lib.INVALID_ARGUMENT
    assert L.cpq_kv_plan(None, *[None] * 3, 0, 0, 16, None, 0, *[None] * 5, 0, None) == _lib.INVALID_ARGUMENT
    assert L.cpq_kv_append(None, None, None, 0, 0, None, 0, 0, None, 0) == _lib.INVALID_ARGUMENT
    assert L.cpq_kv_gather(None, None, None, 0, None, None) == _lib.INVALID_ARGUMENT
    assert L.cpq_kv_attention(None, None, None) == _lib.INVALID_ARGUMENT


def test_buffer_checks():
    """The Python layer's checks come before any call of the library."""
    u32 = lambda n: Buffer(None, None, n, "u32", 4 * n)
    with pytest.raises(TypeError):
        kkv.kv_plan(None, Buffer(None, None, 2, "f32", 8), u32(2), u32(8), 4, 16, u32(8), u32(1), u32(3), u32(2),
                    u32(5), u32(5), u32(1))
    with pytest.raises(_lib.InvalidArgument):
        kkv.kv_plan(None, u32(2), u32(2), u32(7), 4, 16, u32(8), u32(1), u32(3), u32(2), u32(5), u32(5), u32(1))
    with pytest.raises(_lib.InvalidArgument):
        kkv.kv_release(None, u32(1), u32(2), u32(8), 4, 16, u32(8), u32(1), u32(2), u32(1))
    b = Buffer(None, None, 100, "bf16", 512)
    with pytest.raises(_lib.InvalidArgument):
        kkv._attention_args(*[0] * 15, 1.0, 1, -1)
    with pytest.raises(_lib.InvalidArgument):
        kkv._strides("op", "bf16", (50, 10), b, 3, 1, 8)  # 2 * 50 + 8 elements
    assert kkv._strides("op", "bf16", (46, 10), b, 3, 1, 8) == (46, 10)
    view = u32(10)
    view.ptr = 0
    with pytest.raises(ValueError):
        view.slice(5, 6)
    assert len(view.slice(5, 5)) == 5
    view.ptr = None


# ---------------------------------------------------------------------------
# Release and plan
# ---------------------------------------------------------------------------

def model_release(finished, lens, table, bs, free, count):
    free, lens = list(free), list(lens)
    width, lost = table.shape[1], 0
    for s, end in enumerate(finished):
        if end:
            for b in table[s, :min(-(-int(lens[s]) // bs), width)]:
                if count < len(free):
                    free[count] = b
                    count += 1
                else:
                    lost += 1
            lens[s] = 0
    return np.array(free, np.uint32), np.array(lens, np.uint32), count, lost


def model_plan(lens, new, table, bs, free, count, cap):
    """Token by token; a sequence's tokens after one without a place have none."""
    table, width = table.copy(), table.shape[1]
    n_free, lost = min(count, len(free)), 0
    starts, kv, slots, positions = [0], [], [], []
    for s, n in enumerate(new):
        held = min(int(n), cap - len(slots))
        lost += int(n) - held
        placed = min(int(lens[s]), width * bs)
        for p in range(int(lens[s]), int(lens[s]) + held):
            slot = NONE
            if p // bs < width:
                if p // bs < min(-(-int(lens[s]) // bs), width):
                    block = int(table[s, p // bs])
                elif p % bs == 0 and n_free > 0:
                    n_free -= 1
                    block = table[s, p // bs] = int(free[n_free])
                elif p % bs == 0:
                    block = NONE
                if block != NONE:
                    slot = block * bs + p % bs
                    placed = p + 1
            lost += slot == NONE
            slots.append(slot)
            positions.append(p)
        kv.append(placed)
        starts.append(len(slots))
    pad = cap - len(slots)
    u = lambda x: np.array(x, np.uint32)
    return (u(starts), u(kv), u(slots + [NONE] * pad), u(positions + [0] * pad), table, n_free), lost


def _lengths(rng, n, bs, width, most_new):
    lens = rng.integers(0, width * bs // 2, n)
    lens[rng.random(n) < 0.3] = 0
    exact = rng.random(n) < 0.3  # full last blocks
    lens[exact] = lens[exact] // bs * bs
    new = rng.integers(0, most_new + 1, n)
    return lens.astype(np.uint32), new.astype(np.uint32)


def _table(rng, lens, bs, width, spare):
    """Random distinct blocks; (table, free list)."""
    have = [min(-(-int(n) // bs), width) for n in lens]
    ids = rng.permutation(sum(have) + spare).astype(np.uint32)
    table = np.full((len(lens), width), 0xDEAD, np.uint32)
    at = 0
    for s, n in enumerate(have):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, ids[at:]


def run_plan(device, lens, new, table, bs, free, count, cap):
    up = lambda a: device.upload(np.asarray(a, np.uint32).reshape(-1), "u32")
    n = len(lens)
    T = up(table)
    starts, kv, slots, pos, left = (device.alloc_buffer(k, "u32") for k in (n + 1, n, cap, cap, 1))
    cmds = device.commands()
    kkv.kv_plan(cmds, up(lens), up(new), T, table.shape[1], bs, up(free), up([count]), starts, kv, slots, pos, left)
    lost = ""
    try:
        cmds.commit_and_wait()
    except _lib.InvalidArgument as e:
        lost = e.message
    got = (starts.to_numpy(), kv.to_numpy(), slots.to_numpy(), pos.to_numpy(), T.to_numpy().reshape(table.shape),
           int(left.to_numpy()[0]))
    return got, lost


def _same(got, want):
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


@pytest.mark.gpu
@pytest.mark.parametrize("n,bs,width,most_new,extra", [
    (1, 16, 4, 1, 0), (1, 16, 40, 300, 5), (5, 32, 8, 40, 0), (64, 16, 64, 1, 0), (1024, 16, 16, 3, 100),
    (1025, 64, 3, 90, 7), (2500, 16, 4, 12, 0), (8192, 16, 2, 2, 50), (3, 1024, 3, 1500, 1)])
def test_plan(device, n, bs, width, most_new, extra):
    rng = np.random.default_rng(n + bs)
    lens, new = _lengths(rng, n, bs, width, most_new)
    new = np.minimum(new, width * bs - lens).astype(np.uint32)  # rows that hold them
    table, free = _table(rng, lens, bs, width, int(new.sum()) // bs + n + 3)
    cap = int(new.sum()) + extra
    want, lost = model_plan(lens, new, table, bs, free, len(free), cap)
    got, message = run_plan(device, lens, new, table, bs, free, len(free), cap)
    assert lost == 0 and message == ""
    _same(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("n,bs,width,most_new,spare,cut", [
    (4, 16, 4, 60, 3, 0), (40, 16, 6, 90, 20, 300), (7, 32, 2, 100, 100, 1), (1, 16, 3, 200, 0, 0),
    (1500, 16, 3, 30, 400, 5000)])
def test_plan_without_room(device, n, bs, width, most_new, spare, cut):
    """Table rows too short, too few free blocks, fewer slots than tokens."""
    rng = np.random.default_rng(n * 3 + spare)
    lens, new = _lengths(rng, n, bs, width, most_new)
    table, free = _table(rng, lens, bs, width, spare)
    cap = max(0, int(new.sum()) - cut)
    want, lost = model_plan(lens, new, table, bs, free, len(free), cap)
    got, message = run_plan(device, lens, new, table, bs, free, len(free), cap)
    _same(got, want)
    assert (f"{lost} token(s)" in message) if lost else message == ""


@pytest.mark.gpu
def test_plan_of_nothing(device):
    none = np.zeros(0, np.uint32)
    got, message = run_plan(device, none, none, np.zeros((0, 3), np.uint32), 16, np.arange(4), 4, 6)
    assert message == ""
    _same(got, ([0], [], [NONE] * 6, [0] * 6, np.zeros((0, 3)), 4))
    # Lengths past the table, a count past the list, lengths that wrap 32 bits.
    table = np.arange(8, dtype=np.uint32).reshape(2, 4)
    got, message = run_plan(device, [0xFFFFFFF0, 3], [0xFFFFFFFF, 2], table, 16, np.arange(100, 103), 1000, 20)
    assert np.array_equal(got[0], [0, 20, 20])
    assert np.array_equal(got[1], [64, 3]) and np.all(got[2] == NONE) and got[5] == 3
    assert f"{(0xFFFFFFFF - 20 + 2 + 20) % 2**32} token(s)" in message  # cut off, and without a slot


@pytest.mark.gpu
@pytest.mark.parametrize("n,bs,width,spare,cap_short", [(1, 16, 3, 2, 0), (9, 16, 5, 0, 0), (300, 32, 7, 11, 0),
                                                         (2100, 16, 3, 5, 0), (50, 16, 6, 0, 17)])
def test_release(device, n, bs, width, spare, cap_short):
    rng = np.random.default_rng(n)
    lens, _ = _lengths(rng, n, bs, width, 0)
    lens[: n // 7] = width * bs + 5  # longer than the table's rows
    table, free = _table(rng, lens, bs, width, spare)
    finished = (rng.random(n) < 0.5).astype(np.uint32) * 7
    finished[0] = 1
    blocks = sum(min(-(-int(k) // bs), width) for k, f in zip(lens, finished) if f)
    full = np.full(max(0, spare + blocks - cap_short), 0xBEEF, np.uint32)
    full[:spare] = free[:spare]
    want_free, want_lens, count, lost = model_release(finished, lens, table, bs, full, spare)
    up = lambda a: device.upload(np.asarray(a, np.uint32).reshape(-1), "u32")
    F, out, left = up(full), device.alloc_buffer(n, "u32"), device.alloc_buffer(1, "u32")
    cmds = device.commands()
    kkv.kv_release(cmds, up(finished), up(lens), up(table), width, bs, F, up([spare]), out, left)
    if lost:
        with pytest.raises(_lib.InvalidArgument, match=f"{lost} block"):
            cmds.commit_and_wait()
    else:
        cmds.commit_and_wait()
    assert np.array_equal(F.to_numpy(), want_free)
    assert np.array_equal(out.to_numpy(), want_lens)
    assert left.to_numpy()[0] == count


@pytest.mark.gpu
def test_outputs_may_not_overlap(device):
    b = lambda n: device.alloc_buffer(n, "u32")
    lens, count = b(4), b(1)
    cmds = device.commands()
    with pytest.raises(_lib.InvalidArgument, match="overlaps"):
        kkv.kv_plan(cmds, lens, b(4), b(8), 2, 16, b(8), count, b(5), b(4), b(3), b(3), count)
    with pytest.raises(_lib.InvalidArgument, match="overlaps"):
        kkv.kv_release(cmds, b(4), lens, b(8), 2, 16, b(8), count, lens, b(1))


# ---------------------------------------------------------------------------
# Append and gather
# ---------------------------------------------------------------------------

def quantize(x, gs, dtype):
    """The definition in float32, correctly rounded at each step: q, and the
    scale and bias patterns, of x[n, heads, dim] (values of T)."""
    g = x.astype(np.float32).reshape(*x.shape[:2], x.shape[2] // gs, gs)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        lo = np.where((lo == 0) & np.signbit(g).any(-1), np.float32(-0.0), lo)  # -0 lies below 0
        span = (hi - lo).astype(np.float32)
        ok = np.isfinite(span) & np.isfinite(g).all(-1)
        s = np.where(ok, to_bits((np.where(ok, span, 0) / np.float32(15)).astype(np.float32), dtype), 0)
        b = np.where(ok, to_bits(np.where(ok, lo, 0).astype(np.float32), dtype), NAN[dtype])
        sf = from_bits(s.astype(np.uint16), dtype).astype(np.float32)
        q = np.rint(((g - lo[..., None]).astype(np.float32) / sf[..., None]).astype(np.float32)).clip(0, 15)
        q = np.where((ok & (sf != 0))[..., None], q, 0)
    return q.astype(np.uint32).reshape(x.shape), s.astype(np.uint16), b.astype(np.uint16)


def dequantize(q, s, b, gs, dtype):
    """float64."""
    sf, bf = (from_bits(v, dtype).astype(np.float64)[..., None] for v in (s, b))
    return (q.reshape(*s.shape, gs) * sf + bf).reshape(q.shape)


class Host:
    """A cache's four arrays on the host, filled with what nobody may read."""

    def __init__(self, rng, dtype, n_blocks, bs, heads, dim, gs):
        self.dtype, self.bs, self.gs, self.dim, self.heads, self.n = dtype, bs, gs, dim, heads, n_blocks
        W, G = dim // 8, dim // gs
        self.k_q = rng.integers(0, 2**32, (n_blocks, heads, bs, W), dtype=np.uint32)
        self.v_q = rng.integers(0, 2**32, (n_blocks, heads, bs // 4, W, 4), dtype=np.uint32)
        nan = np.uint32(NAN[dtype] * 0x10001)
        self.k_sb = np.full((n_blocks, heads, bs, G), nan)
        self.v_sb = np.full((n_blocks, heads, bs // 4, G, 4), nan)

    def put(self, slots, k, v):
        """k, v: (q, s, b) of as many rows as there are slots."""
        for which, (q, s, b) in (("k", k), ("v", v)):
            words = np.zeros((*q.shape[:2], self.dim // 8), np.uint32)
            for j in range(8):
                words |= q[:, :, j::8] << np.uint32(4 * j)
            sb = s.astype(np.uint32) | b.astype(np.uint32) << np.uint32(16)
            for i, slot in enumerate(np.asarray(slots).tolist()):
                if slot >= self.n * self.bs:
                    continue
                blk, off = slot // self.bs, slot % self.bs
                if which == "k":
                    self.k_q[blk, :, off], self.k_sb[blk, :, off] = words[i], sb[i]
                else:
                    self.v_q[blk, :, off // 4, :, off % 4] = words[i]
                    self.v_sb[blk, :, off // 4, :, off % 4] = sb[i]

    def arrays(self):
        return self.k_q, self.k_sb, self.v_q, self.v_sb

    def upload(self, device):
        return kkv.KvCache(device, self.dtype, self.n, self.bs, self.heads, self.dim, self.gs,
                           buffers=[device.upload(a.reshape(-1), "u32") for a in self.arrays()])


def _rows(rng, n, heads, dim, dtype, size=1.0):
    x = rng.standard_normal((n, heads, dim)) * size * np.exp(rng.standard_normal((heads, dim)) * 0.4)
    bits = to_bits(x.astype(np.float32), dtype)
    return bits, from_bits(bits, dtype).astype(np.float32)


GEOMETRIES = [("bf16", 64, 32, 16), ("bf16", 64, 64, 32), ("f16", 128, 32, 16), ("bf16", 128, 64, 64),
              ("f16", 128, 128, 16), ("bf16", 256, 32, 16), ("f16", 256, 64, 1024), ("bf16", 256, 128, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", GEOMETRIES)
@pytest.mark.parametrize("tokens,heads", [(1, 1), (7, 3), (70, 2)])
def test_append_gather(device, dtype, dim, gs, bs, tokens, heads):
    """Words and constants bit for bit, neighbours untouched; padding and bad
    slots; strided sources; the gather of what was written and of padding."""
    rng = np.random.default_rng(dim + gs + tokens)
    n = -(-tokens // bs) + 3
    host = Host(rng, dtype, n, bs, heads, dim, gs)
    cache = host.upload(device)
    kb, kx = _rows(rng, tokens, heads, dim, dtype)
    vb, vx = _rows(rng, tokens, heads, dim, dtype, 0.02)
    slots = rng.permutation(n * bs)[:tokens].astype(np.uint32)
    if tokens > 20:  # consecutive slots too
        slots[8:20] = np.setdiff1d(np.arange(n * bs), np.concatenate([slots[:8], slots[20:]]))[:12]
        slots[3] = NONE
        slots[5] = n * bs
        slots[6] = 0xFFFFFFF0
    # Rows of a fused projection: [tokens, 1 + 2 * heads, dim], keys then values behind one other head.
    fused = np.zeros((tokens, 1 + 2 * heads, dim), np.uint16)
    fused[:, 1:1 + heads], fused[:, 1 + heads:] = kb, vb
    X = device.upload(fused.reshape(-1), dtype)
    S = device.upload(slots, "u32")
    strides = ((1 + 2 * heads) * dim, dim)
    cmds = device.commands()
    kkv.kv_append(cmds, cache, X.slice(dim, len(X) - dim), X.slice((1 + heads) * dim, len(X) - (1 + heads) * dim), S,
                  tokens, k_strides=strides, v_strides=strides)
    if tokens > 20:
        with pytest.raises(_lib.InvalidArgument, match="2 slot"):
            cmds.commit_and_wait()
    else:
        cmds.commit_and_wait()
    k, v = quantize(kx, gs, dtype), quantize(vx, gs, dtype)
    host.put(slots, k, v)
    for name, want in zip(("k_q", "k_sb", "v_q", "v_sb"), host.arrays()):
        assert np.array_equal(getattr(cache, name).to_numpy().reshape(want.shape), want), name
    outs = [device.alloc_buffer(tokens * heads * dim, dtype) for _ in range(2)]
    kkv.kv_gather(cmds, cache, S, tokens, *outs)
    if tokens > 20:
        with pytest.raises(_lib.InvalidArgument, match="2 slot"):
            cmds.commit_and_wait()
    else:
        cmds.commit_and_wait()
    live = slots < n * bs
    for out, (q, s, b) in zip(outs, (k, v)):
        want = to_bits(dequantize(q, s, b, gs, dtype).astype(np.float32), dtype)
        want[~live] = 0
        assert np.array_equal(out.to_numpy().reshape(want.shape), want)
    # One output alone.
    only = [device.upload(np.full(tokens * heads * dim, 0x5555, np.uint16), dtype) for _ in range(2)]
    good = device.upload(np.where(live, slots, NONE).astype(np.uint32), "u32")
    kkv.kv_gather(cmds, cache, good, tokens, only[0], None)
    kkv.kv_gather(cmds, cache, good, tokens, None, only[1])
    cmds.commit_and_wait()
    for a, b in zip(only, outs):
        assert np.array_equal(a.to_numpy(), b.to_numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_append_special_values(device, dtype):
    """Constant groups, Inf, NaN, ranges that overflow, tiny ranges, ties."""
    dim, gs, bs = 128, 32, 16
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 1, dim)).astype(np.float32)
    x[0, 0, :32] = 0.75
    x[1, 0, 40] = np.inf
    x[2, 0, 70] = -np.inf
    x[3, 0, 127] = np.nan
    x[4] = np.nan
    x[5, 0, :32] = np.where(np.arange(32) % 2, 1, -1) * (3.3e38 if dtype == "bf16" else 65504.0)  # f16: no overflow
    x[6] *= 1e-38 if dtype == "bf16" else 1e-6
    x[7, 0] = (np.arange(dim) % 31) * 0.125  # halves of a step: ties
    x[8, 0] = -0.0
    x[9, 0, ::2] = 0.0
    x[10, 0] = np.arange(dim) * 2.0 ** -8
    bits = to_bits(x, dtype)
    xt = from_bits(bits, dtype).astype(np.float32)
    host = Host(rng, dtype, 1, bs, 1, dim, gs)
    cache = host.upload(device)
    X, S = device.upload(bits.reshape(-1), dtype), device.upload(np.arange(12, dtype=np.uint32), "u32")
    cmds = device.commands()
    kkv.kv_append(cmds, cache, X, X, S, 12)
    outs = [device.alloc_buffer(12 * dim, dtype) for _ in range(2)]
    kkv.kv_gather(cmds, cache, S, 12, *outs)
    cmds.commit_and_wait()
    q, s, b = quantize(xt, gs, dtype)
    want = dequantize(q, s, b, gs, dtype).astype(np.float32)
    for out in outs:
        got = from_bits(out.to_numpy(), dtype).astype(np.float32).reshape(want.shape)
        ref = from_bits(to_bits(want, dtype), dtype).astype(np.float32)
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert np.array_equal(got[~np.isnan(got)], ref[~np.isnan(ref)])
    assert np.isnan(want[1, 0, 32:64]).all() and np.isfinite(want[1, 0, 64:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,low,high", [("bf16", -132, 122), ("f16", -22, 10)])
def test_append_near_halves(device, dtype, low, high):
    """Values next to half steps, over the type's whole range: bit for bit."""
    dim, gs, bs, n = 128, 32, 64, 2048
    rng = np.random.default_rng(17)
    span = np.exp2(rng.uniform(low, high, (n, dim // gs, 1)))
    base = rng.choice([0.0, 1.0, -1.0, -0.3], (n, dim // gs, 1)) * span * rng.choice([1, 0.01], (n, dim // gs, 1))
    step = rng.integers(0, 31, (n, dim // gs, gs)) / 30.0
    step[..., 0], step[..., 5] = 0.0, 1.0
    bits = to_bits((base + span * step).astype(np.float32).reshape(n, 1, dim), dtype)
    near = bits.astype(np.int64) + rng.integers(-1, 2, bits.shape)  # a unit of T off
    bits = np.where((bits & 0x7FFF) > 0, near, bits).astype(np.uint16)
    x = from_bits(bits, dtype).astype(np.float32)
    assert np.isfinite(x).all()
    host = Host(rng, dtype, n // bs, bs, 1, dim, gs)
    cache = host.upload(device)
    X, S = device.upload(bits.reshape(-1), dtype), device.upload(np.arange(n, dtype=np.uint32), "u32")
    cmds = device.commands()
    kkv.kv_append(cmds, cache, X, X, S, n)
    cmds.commit_and_wait()
    want = quantize(x, gs, dtype)
    host.put(np.arange(n), want, want)
    for name, w in zip(("k_q", "k_sb", "v_q", "v_sb"), host.arrays()):
        assert np.array_equal(getattr(cache, name).to_numpy().reshape(w.shape), w), name


@pytest.mark.gpu
def test_nothing_to_append(device):
    cache = Host(np.random.default_rng(0), "bf16", 2, 16, 1, 64, 32).upload(device)
    before = [getattr(cache, n).to_numpy() for n in ("k_q", "k_sb", "v_q", "v_sb")]
    x, s = device.alloc_buffer(64, "bf16"), device.alloc_buffer(1, "u32")
    cmds = device.commands()
    kkv.kv_append(cmds, cache, x, x, s, 0)
    kkv.kv_gather(cmds, cache, s, 0, x, x)
    kkv.kv_gather(cmds, cache, s, 1, None, None)
    with pytest.raises(_lib.InvalidArgument):
        kkv.kv_append(cmds, cache, x, x, s, 1, k_strides=(4, 4))
    with pytest.raises(_lib.InvalidArgument):
        kkv.kv_append(cmds, cache, x.slice(4, 60), x, s, 1, k_strides=(0, 0))
    cmds.commit_and_wait()
    for n, b in zip(("k_q", "k_sb", "v_q", "v_sb"), before):
        assert np.array_equal(getattr(cache, n).to_numpy(), b)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

class Batch:
    """Sequences with their cache on host and device, and their queries."""

    def __init__(self, rng, device, dtype, dim, gs, bs, kv_heads, group, q_lens, kv_lens, sharp=1.0):
        self.dtype, self.dim, self.group, self.kv_heads = dtype, dim, group, kv_heads
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        self.device, self.heads = device, kv_heads * group
        self.width = max([-(-n // bs) for n in kv_lens] + [0]) + 1
        used = sum(-(-n // bs) for n in kv_lens)
        host = Host(rng, dtype, used + 2, bs, kv_heads, dim, gs)
        order = rng.permutation(used + 2)
        self.table = np.full((len(kv_lens), self.width), 0xFFFFFFFF, np.uint32)
        self.k, self.v, at = [], [], 0
        for i, n in enumerate(kv_lens):
            m = -(-n // bs)
            self.table[i, :m] = order[at:at + m]
            at += m
            _, kx = _rows(rng, n, kv_heads, dim, dtype, 0.8)
            _, vx = _rows(rng, n, kv_heads, dim, dtype, 0.7)
            kq, vq = quantize(kx, gs, dtype), quantize(vx, gs, dtype)
            j = np.arange(n)
            host.put(self.table[i][j // bs] * bs + j % bs, kq, vq)
            self.k.append(dequantize(*kq, gs, dtype))
            self.v.append(dequantize(*vq, gs, dtype))
        self.host = host
        self.starts = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.uint32)
        self.tokens = int(self.starts[-1])
        q = rng.standard_normal((self.tokens, self.heads, dim)) * sharp
        self.q_bits = to_bits(q.astype(np.float32), dtype)
        self.q = from_bits(self.q_bits, dtype).astype(np.float64)

    def run(self, causal=True, window=0, cmds=None, max_q=None, max_kv=None, fused=0, heads_first=False, scale=None,
            cache=None):
        """Output bits [tokens, heads, dim]; fused: other heads in q's rows."""
        d, n = self.device, self.tokens
        up = lambda a: d.upload(np.asarray(a, np.uint32).reshape(-1), "u32")
        rows = np.zeros((n, self.heads + fused, self.dim), np.uint16)
        rows[:, :self.heads] = self.q_bits
        out = d.upload(np.full(n * self.heads * self.dim, 0x5A5A, np.uint16), self.dtype)
        cmds = cmds or d.commands()
        self.keep = (cache or self.host.upload(d), d.upload(rows.reshape(-1), self.dtype), up(self.table),
                     up(self.starts), up(self.kv_lens), out)
        kkv.kv_attention(cmds, *self.keep[:3], self.width, *self.keep[3:], n, self.heads, len(self.kv_lens),
                         max(self.q_lens) if max_q is None else max_q,
                         max(self.kv_lens) if max_kv is None else max_kv, scale or self.dim ** -0.5, causal=causal,
                         window=window, q_strides=((self.heads + fused) * self.dim, self.dim),
                         out_strides=(self.dim, n * self.dim) if heads_first else None)
        cmds.commit_and_wait()
        got = out.to_numpy()
        return got.reshape(self.heads, n, self.dim).transpose(1, 0, 2) if heads_first else \
            got.reshape(n, self.heads, self.dim)

    def expect(self, causal=True, window=0, scale=None):
        """(out, bound of the internal error) in float64.  Operands are rounded
        to f16 at most (half a unit 2^-12, relative): a logit is off by at most
        2^-11 of the sum of its terms' sizes, a weight by twice that (numerator
        and sum), by its own rounding and its value's."""
        scale = scale or self.dim ** -0.5
        out, bound = np.zeros(self.q.shape), np.zeros(self.q.shape)
        for i, (m, n) in enumerate(zip(self.q_lens, self.kv_lens)):
            pos, j = np.arange(n - m, n)[:, None], np.arange(n)[None, :]
            seen = np.ones((m, n), bool)
            if causal:
                seen &= j <= pos
            if window:
                seen &= j > pos - window
            for h in range(self.heads if m and n else 0):
                q = self.q[self.starts[i]:self.starts[i + 1], h]
                k, v = self.k[i][:, h // self.group], self.v[i][:, h // self.group]
                z = np.where(seen, q @ k.T * scale, -np.inf)
                top = z.max(1, keepdims=True)
                p = np.exp(z - np.where(np.isfinite(top), top, 0))
                total = p.sum(1, keepdims=True)
                p /= np.where(total == 0, 1, total)
                size = np.where(seen, np.abs(q) @ np.abs(k).T * scale, 0).max(1, keepdims=True)
                out[self.starts[i]:self.starts[i + 1], h] = p @ v
                bound[self.starts[i]:self.starts[i + 1], h] = (2.0 ** -10 * size + 2.0 ** -10) * (p @ np.abs(v))
        return out, bound

    def check(self, bits, causal=True, window=0, scale=None):
        want, bound = self.expect(causal, window, scale)
        got = from_bits(bits, self.dtype).astype(np.float64)
        assert np.isfinite(got).all()
        unit = 2.0 ** -9 if self.dtype == "bf16" else 2.0 ** -12
        err = np.abs(got - want)
        limit = unit * 1.02 * np.abs(want) + bound + 1e-7
        assert (err <= limit).all(), (err - limit).max()
        # A rounding's root mean square is 0.58 of half a unit; operands add up to as much again in f16.
        assert np.linalg.norm(err) <= (2.2e-3 if self.dtype == "bf16" else 9e-4) * np.linalg.norm(want) + 1e-7


def _close(got, want, dtype):
    """Equal but for a rounding and what operands keep of their tile's largest."""
    a, b = (from_bits(x, dtype).astype(np.float64) for x in (got, want))
    unit = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -10
    return bool((np.abs(a - b) <= unit * np.abs(b) + 2.0 ** -16 * np.abs(b).max(initial=0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", GEOMETRIES)
@pytest.mark.parametrize("group", [1, 4, 7])
def test_one_token(device, dtype, dim, gs, bs, group):
    """Single queries over every length around a tile's and a block's end."""
    rng = np.random.default_rng(dim * gs + group)
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 300]
    b = Batch(rng, device, dtype, dim, gs, bs, 2, group, [1] * len(kv), kv)
    b.check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,bs", GEOMETRIES)
@pytest.mark.parametrize("group,causal,window", [(1, True, 0), (4, False, 0), (3, True, 37), (8, True, 0),
                                                 (2, False, 70)])
def test_queries(device, dtype, dim, gs, bs, group, causal, window):
    """Many queries of several sequences, with cached keys before them or none."""
    rng = np.random.default_rng(dim + gs + group)
    q, kv = [1, 40, 0, 130, 3, 65], [77, 40, 50, 200, 3, 129]
    b = Batch(rng, device, dtype, dim, gs, bs, 2, group, q, kv)
    b.check(b.run(causal, window), causal, window)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 5, 16, 20, 40])
@pytest.mark.parametrize("queries", [1, 2, 9])
def test_groups(device, group, queries):
    """Odd and large groups of heads on one key/value head."""
    rng = np.random.default_rng(group * 10 + queries)
    b = Batch(rng, device, "bf16", 128, 64, 16, 1, group, [queries, queries], [90, 300])
    b.check(b.run())


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q", [1, 30, 100])
def test_empty_rows(device, causal, q):
    """No keys at all, and more queries than keys: rows before the first key
    are zero where causal."""
    rng = np.random.default_rng(q)
    b = Batch(rng, device, "f16", 64, 32, 16, 1, 2, [q, q, q], [0, q // 2, q])
    out = b.run(causal)
    b.check(out, causal)
    assert not out[:q].any()
    if causal:
        assert not out[q:q + q - q // 2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 5, 70])
def test_long(device, q):
    """Keys split over workgroups, on both sides of what one takes."""
    rng = np.random.default_rng(q)
    b = Batch(rng, device, "bf16", 128, 64, 32, 1, 4, [q, q, q], [2049, 5000, 900])
    first = b.run()
    b.check(first)
    assert np.array_equal(b.run(), first)  # same bits again
    b.check(b.run(window=1500), window=1500)
    b.check(b.run(max_kv=100))  # the bound only steers the split
    b.check(b.run(max_kv=100000))


@pytest.mark.gpu
@pytest.mark.parametrize("sharp,scale", [(30.0, None), (1.0, 1e-6), (1000.0, 0.05), (1e-4, 20.0)])
def test_logit_ranges(device, sharp, scale):
    """Weights on one key, flat weights, large and tiny queries."""
    rng = np.random.default_rng(3)
    for dtype in ("bf16", "f16"):
        b = Batch(rng, device, dtype, 128, 64, 16, 1, 3, [1, 40], [500, 77], sharp=sharp)
        want, bound = b.expect(scale=scale)
        got = from_bits(b.run(scale=scale), dtype).astype(np.float64)
        unit = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
        assert (np.abs(got - want) <= unit * 1.02 * np.abs(want) + bound + 1e-7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,k_size,v_size", [("bf16", 1e4, 1e6), ("bf16", 1e-8, 1e-12), ("bf16", 1.0, 1e30),
                                                 ("f16", 50.0, 4000.0), ("f16", 1e-3, 1e-5)])
def test_value_ranges(device, dtype, k_size, v_size):
    """Keys and values far from 1, and rows of very different sizes in one tile."""
    rng = np.random.default_rng(8)
    b = Batch(rng, device, dtype, 128, 64, 16, 1, 4, [1, 30], [200, 60])
    for i, n in enumerate(b.kv_lens):
        step = np.exp(rng.standard_normal((n, 1, 1)))
        j = np.arange(n)
        parts = []
        for size in (k_size, v_size):
            x = rng.standard_normal((n, 1, 128)) * step * size
            x = x.clip(-6e4, 6e4) if dtype == "f16" else x  # finite in T
            parts.append(quantize(from_bits(to_bits(x.astype(np.float32), dtype), dtype).astype(np.float32), 64, dtype))
        b.host.put(b.table[i][j // 16] * 16 + j % 16, *parts)
        b.k[i], b.v[i] = (dequantize(*p, 64, dtype) for p in parts)
    scale = 128 ** -0.5 / k_size
    want, bound = b.expect(scale=scale)
    got = from_bits(b.run(scale=scale), dtype).astype(np.float64)
    unit = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0  # subnormal outputs
    # Operands keep 2^-19 of the largest in their tile.
    largest = max(np.abs(v).max() for v in b.v)
    assert (np.abs(got - want) <= unit * 1.02 * np.abs(want) + bound + 2.0 ** -18 * largest + tiny).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 40])
@pytest.mark.parametrize("n,sizes", [
    (20, (1e-8, 1e-8, 1e-8, 1e-8)),     # less than a tile
    (64, (1e-6, 1e4, 1e4, 1e4)), (64, (1e4, 1e-6, 1e-6, 1e-6)), (130, (1e-3, 1.0, 1e3, 1e-3)),
    (100, (0.0, 1.0, 1.0, 0.0)), (40, (0.0, 0.0, 0.0, 0.0)), (140, (1.0, 1e-30, 1e30, 0.0))])
def test_value_sizes_apart(device, q, n, sizes):
    """Runs of 16 keys whose values' sizes differ, zeros among them: weights of
    tiny or zero values still count in the sum."""
    rng = np.random.default_rng(n)
    b = Batch(rng, device, "bf16", 128, 64, 16, 1, 4, [q], [n])
    j = np.arange(n)
    x = rng.standard_normal((n, 1, 128)) * np.array(sizes)[j // 16 % 4][:, None, None]
    parts = quantize(from_bits(to_bits(x.astype(np.float32), "bf16"), "bf16").astype(np.float32), 64, "bf16")
    kx = _rows(rng, n, 1, 128, "bf16", 0.8)[1]
    keys = quantize(kx, 64, "bf16")
    b.host.put(b.table[0][j // 16] * 16 + j % 16, keys, parts)
    b.k[0], b.v[0] = dequantize(*keys, 64, "bf16"), dequantize(*parts, 64, "bf16")
    want, bound = b.expect(causal=False)
    got = from_bits(b.run(causal=False), "bf16").astype(np.float64)
    largest = np.abs(b.v[0]).max()
    assert (np.abs(got - want) <= 2.0 ** -9 * 1.02 * np.abs(want) + bound + 2.0 ** -18 * largest).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs", [("bf16", 64, 32), ("f16", 64, 64), ("bf16", 256, 128), ("f16", 256, 32),
                                          ("f16", 128, 128)])
def test_prompt_values_apart(device, dtype, dim, gs):
    """Prompts whose values' sizes rise and fall by 10^3 from run to run, in every
    width, whole and split."""
    rng = np.random.default_rng(dim + gs)
    for q, n in ((90, 90), (40, 700), (300, 333)):
        b = Batch(rng, device, dtype, dim, gs, 16, 1, 3, [q], [n])
        j = np.arange(n)
        size = np.array((1.0, 1e-3, 30.0, 0.0, 1e-2, 1.0, 0.0))[j // 16 % 7]
        x = rng.standard_normal((n, 1, dim)) * size[:, None, None]
        vq = quantize(from_bits(to_bits(x.astype(np.float32), dtype), dtype).astype(np.float32), gs, dtype)
        kq = quantize(_rows(rng, n, 1, dim, dtype, 0.8)[1], gs, dtype)
        b.host.put(b.table[0][j // 16] * 16 + j % 16, kq, vq)
        b.k[0], b.v[0] = dequantize(*kq, gs, dtype), dequantize(*vq, gs, dtype)
        unit = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
        for causal in (True, False):
            want, bound = b.expect(causal=causal)
            got = from_bits(b.run(causal=causal), dtype).astype(np.float64)
            assert (np.abs(got - want) <= unit * 1.02 * np.abs(want) + bound + 2.0 ** -18 * np.abs(b.v[0]).max()).all()


def _prompts(rng, device, dtype, gs):
    """Enough row tiles for workgroups of eight waves: 34 prompts over 8 heads."""
    q = rng.integers(6, 60, 34)
    kv = q + rng.integers(0, 500, 34)
    q[3], kv[3], kv[4], q[5], kv[5] = 130, 130, q[4], 200, 1200
    return Batch(rng, device, dtype, 128, gs, 16, 8, 3, q.tolist(), kv.tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gs,causal,window", [("bf16", 64, True, 0), ("f16", 32, False, 0), ("f16", 128, True, 70),
                                                    ("bf16", 32, True, 333)])
def test_many_prompts(device, dtype, gs, causal, window):
    b = _prompts(np.random.default_rng(gs), device, dtype, gs)
    first = b.run(causal, window)
    b.check(first, causal, window)
    assert np.array_equal(b.run(causal, window), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gs", [("bf16", 64), ("f16", 32)])
def test_many_prompts_values_apart(device, dtype, gs):
    """Values of very different sizes in neighbouring runs of 16, and what no row
    may see after every sequence's end not finite."""
    rng = np.random.default_rng(gs + 1)
    b = _prompts(rng, device, dtype, gs)
    for i, n in enumerate(b.kv_lens):
        j = np.arange(n)
        size = np.array((1.0, 1e-3, 30.0, 0.0, 1e-2, 1.0, 0.0))[(j // 16 + i) % 7]
        x = rng.standard_normal((n, 8, 128)) * size[:, None, None]
        vq = quantize(from_bits(to_bits(x.astype(np.float32), dtype), dtype).astype(np.float32), gs, dtype)
        kq = quantize(_rows(rng, n, 8, 128, dtype, 0.8)[1], gs, dtype)
        b.host.put(b.table[i][j // 16] * 16 + j % 16, kq, vq)
        b.k[i], b.v[i] = dequantize(*kq, gs, dtype), dequantize(*vq, gs, dtype)
    want, bound = b.expect()
    got = from_bits(b.run(), dtype).astype(np.float64)
    unit = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
    largest = max(np.abs(v).max() for v in b.v)
    assert (np.abs(got - want) <= unit * 1.02 * np.abs(want) + bound + 2.0 ** -18 * largest).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,gs,group", [(64, 64, 4), (128, 64, 4), (256, 64, 2)])
def test_long_token_beside_a_prompt(device, dim, gs, group):
    """A single token over keys in many parts, beside a prompt and a draft."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, device, "bf16", dim, gs, 32, 1, group, [1, 150, 3], [9001, 170, 4500])
    first = b.run()
    b.check(first)
    assert np.array_equal(b.run(), first)


@pytest.mark.gpu
def test_many_sequences(device):
    """More sequences than a wave has lanes, lengths of zero among them, one and
    several queries each."""
    rng = np.random.default_rng(11)
    kv = rng.integers(0, 90, 150)
    kv[::17] = 0
    for q in (np.minimum(kv, 1), np.minimum(kv, rng.integers(0, 30, 150))):
        b = Batch(rng, device, "bf16", 64, 32, 16, 2, 3, q.tolist(), kv.tolist())
        b.check(b.run())


@pytest.mark.gpu
def test_many_sequences_some_long(device):
    """Of 140 sequences two are split over workgroups."""
    rng = np.random.default_rng(12)
    kv = rng.integers(1, 40, 140)
    kv[70], kv[139] = 3001, 1700
    for q in (np.ones(140, int), np.minimum(kv, rng.integers(0, 4, 140))):
        b = Batch(rng, device, "f16", 64, 64, 16, 1, 4, q.tolist(), kv.tolist())
        first = b.run()
        b.check(first)
        assert np.array_equal(b.run(), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs,group,q,n", [("bf16", 64, 32, 7, 1, 9000), ("f16", 64, 64, 1, 3, 4200),
                                                    ("bf16", 128, 64, 4, 1, 12345), ("f16", 128, 32, 2, 9, 6000),
                                                    ("bf16", 256, 128, 1, 1, 5001), ("f16", 256, 64, 8, 4, 7000)])
def test_one_long_sequence(device, dtype, dim, gs, group, q, n):
    """More parts than one workgroup joins, beside a sequence of one part and one
    without keys that any row sees."""
    rng = np.random.default_rng(n)
    b = Batch(rng, device, dtype, dim, gs, 32, 1, group, [q, q, 0], [n, q, 0])
    first = b.run()
    b.check(first)
    assert np.array_equal(b.run(), first)
    b.check(b.run(window=4500), window=4500)


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 40])
def test_masked_poison(device, q):
    """Inf and NaN keys and values that no row may see: future tokens, tokens
    outside the window, what a block holds past the sequence's end."""
    rng = np.random.default_rng(q)
    b = Batch(rng, device, "bf16", 128, 64, 16, 2, 4, [q, q], [100, 57])
    b.check(b.run(window=20), window=20)
    for i, n in enumerate(b.kv_lens):
        for p in range(0, n - q - 19):  # before every row's window
            slot = b.table[i, p // 16] * 16 + p % 16
            blk, off = slot // 16, slot % 16
            b.host.k_sb[blk, :, off] = 0x7F80FF80
            b.host.v_sb[blk, :, off // 4, :, off % 4] = 0x7FC07F80
    b.check(b.run(window=20), window=20)
    # A poisoned newest token: causal rows before it stay as they were, its own row is not finite.
    c = Batch(rng, device, "bf16", 128, 64, 16, 2, 4, [q + 2], [90])
    clean = c.run()
    slot = int(c.table[0, 89 // 16]) * 16 + 89 % 16
    c.host.k_sb[slot // 16, :, slot % 16] = 0x7FC07FC0
    c.host.v_sb[slot // 16, :, slot % 16 // 4, :, slot % 4] = 0x7FC07FC0
    got = c.run()
    assert _close(got[:-1], clean[:-1], "bf16")
    assert np.isnan(from_bits(got[-1], "bf16")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 50])
def test_value_poison_stays_in_its_group(device, q):
    """A value group that is Inf or NaN reaches its own dimensions only."""
    rng = np.random.default_rng(q)
    b = Batch(rng, device, "bf16", 128, 64, 16, 1, 4, [q], [120])
    clean = b.run()
    slot = int(b.table[0, 0]) * 16  # key 0: every row sees it
    for pattern in (0x7FC00000, 0x3F807F80, 0xFF800000):
        b.host.v_sb[slot // 16, 0, 0, 1, 0] = pattern
        got = b.run()
        assert _close(got[:, :, :64], clean[:, :, :64], "bf16")
        assert not np.isfinite(from_bits(got[:, :, 64:], "bf16")).any()


@pytest.mark.gpu
def test_layouts_streams_and_graph(device):
    """Queries as slices of wider rows, outputs heads first, another session,
    a captured graph replayed with eager work in between."""
    rng = np.random.default_rng(1)
    for q, kv in (([1, 1, 1], [40, 700, 5]), ([30, 1, 90], [40, 700, 90])):
        b = Batch(rng, device, "f16", 128, 64, 16, 2, 3, q, kv)
        want = b.run()
        assert np.array_equal(b.run(fused=5), want)
        assert np.array_equal(b.run(heads_first=True), want)
        cmds = device.commands()
        b.run(cmds=cmds)
        cache, Q, T, S, L, out = b.keep
        def encode():
            kkv.kv_attention(cmds, cache, Q, T, b.width, S, L, out, b.tokens, b.heads, len(kv), max(q), max(kv),
                             128 ** -0.5, q_strides=(b.heads * 128, 128))
        cmds.begin_capture()
        encode()
        graph = cmds.end_capture()
        for _ in range(3):
            out.write(np.zeros(len(out), np.uint16))
            graph.launch(cmds)
            cmds.wait()
            assert np.array_equal(out.to_numpy().reshape(want.shape), want)
            encode()
            cmds.wait()


@pytest.mark.gpu
def test_bounds_at_their_ends(device):
    """max_q, max_kv and window of zero, and as large as their type."""
    rng = np.random.default_rng(4)
    top = 2 ** 64 - 1
    for q in ([1, 1], [3, 40]):
        b = Batch(rng, device, "bf16", 128, 64, 16, 2, 4, q, [70, 300])
        want = b.run()
        for over in (dict(max_q=top), dict(max_q=2 ** 62), dict(max_kv=top), dict(max_kv=0), dict(window=top),
                     dict(window=2 ** 63), dict(window=2 ** 31 + 5), dict(max_q=top, max_kv=top, window=top)):
            b.check(b.run(**over))
        b.check(b.run(window=301))
        with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
            b.run(max_q=0)
        assert np.all(b.keep[-1].to_numpy() == 0x5A5A)  # not computed
        assert np.array_equal(b.run(), want)


@pytest.mark.gpu
def test_bad_lengths_and_blocks(device):
    """What the device finds wrong is masked or left out, and reported."""
    rng = np.random.default_rng(2)
    b = Batch(rng, device, "bf16", 64, 32, 16, 1, 2, [1, 3, 1], [50, 64, 33])
    run = lambda **over: b.run(max_kv=64, **over)
    want = run()
    for q_max in (1, 2):
        with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
            run(max_q=q_max)
        got = b.keep[-1].to_numpy().reshape(want.shape)
        assert _close(got[[0, 4]], want[[0, 4]], "bf16")
        assert np.all(got[1:4] == 0x5A5A)  # not computed
    table = b.table.copy()
    b.table[2, 1] = 0x7FFFFFFF
    with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
        run()
    got = b.keep[-1].to_numpy().reshape(want.shape)
    assert _close(got[:4], want[:4], "bf16")
    b.table = table
    b.kv_lens[0] = 16 * b.width + 7
    with pytest.raises(_lib.InvalidArgument, match="kv_attention"):
        run()
    got = b.keep[-1].to_numpy().reshape(want.shape)
    assert _close(got[1:], want[1:], "bf16")
    b.kv_lens[0] = 50
    assert np.array_equal(run(), want)


@pytest.mark.gpu
def test_offsets_past_32_bits(device):
    """Blocks whose words lie past 4 GiB in their buffer."""
    rng = np.random.default_rng(4)
    dim, heads, bs, n = 256, 8, 1024, 4200  # 1 MiB of words per block
    cache = kkv.KvCache(device, "bf16", n, bs, heads, dim, 128)
    assert cache.k_q.byte_len > 1 << 32
    kv = 70
    kb, kx = _rows(rng, kv, heads, dim, "bf16", 0.8)
    vb, vx = _rows(rng, kv, heads, dim, "bf16", 0.7)
    slots = (n - 1) * bs + np.arange(kv)
    b = Batch(rng, device, "bf16", dim, 128, bs, heads, 2, [1, 20], [kv, kv])
    b.table[:, 0] = n - 1
    cmds = device.commands()
    S = device.upload(slots.astype(np.uint32), "u32")
    kkv.kv_append(cmds, cache, device.upload(kb.reshape(-1), "bf16"), device.upload(vb.reshape(-1), "bf16"), S, kv)
    outs = [device.alloc_buffer(kv * heads * dim, "bf16") for _ in range(2)]
    kkv.kv_gather(cmds, cache, S, kv, *outs)
    cmds.commit_and_wait()
    for i, (out, x) in enumerate(zip(outs, (kx, vx))):
        parts = quantize(x, 128, "bf16")
        want = dequantize(*parts, 128, "bf16")
        assert np.array_equal(out.to_numpy().reshape(want.shape), to_bits(want.astype(np.float32), "bf16"))
        (b.k if i == 0 else b.v)[:] = [want, want]
    b.check(b.run(cache=cache))


@pytest.mark.gpu
def test_serving_steps(device):
    """The operators together: prompts, then decoded tokens of three requests,
    one of which ends while a fourth arrives; each step's attention over the
    cache as planned equals float64 over the rows gathered back."""
    rng = np.random.default_rng(6)
    dtype, dim, gs, bs, heads, group, width, n_blocks = "bf16", 64, 32, 16, 2, 3, 8, 24
    cache = kkv.KvCache(device, dtype, n_blocks, bs, heads, dim, gs)
    up = lambda a: device.upload(np.asarray(a, np.uint32).reshape(-1), "u32")
    table, free = up(np.full((4, width), NONE)), up(rng.permutation(n_blocks))
    lens, count = up([0, 0, 0, 0]), up([n_blocks])
    steps = [([30, 16, 1, 0], [0] * 4), ([1, 1, 1, 0], [0] * 4), ([1, 0, 1, 45], [0, 1, 0, 0]), ([1, 5, 1, 1], [0] * 4)]
    total = [0, 0, 0, 0]
    cmds = device.commands()
    for new, finished in steps:
        cap = sum(new) + 2
        lens2, count2, starts, kv, slots, pos, count3 = (device.alloc_buffer(k, "u32") for k in (4, 1, 5, 4, cap, cap, 1))
        k, v, q = (_rows(rng, cap, h, dim, dtype)[0] for h in (heads, heads, heads * group))
        Q, out = device.upload(q.reshape(-1), dtype), device.alloc_buffer(cap * heads * group * dim, dtype)
        kkv.kv_release(cmds, up(finished), lens, table, width, bs, free, count, lens2, count2)
        kkv.kv_plan(cmds, lens2, up(new), table, width, bs, free, count2, starts, kv, slots, pos, count3)
        kkv.kv_append(cmds, cache, device.upload(k.reshape(-1), dtype), device.upload(v.reshape(-1), dtype), slots, cap)
        kkv.kv_attention(cmds, cache, Q, table, width, starts, kv, out, cap, heads * group, 4, max(new), width * bs,
                         dim ** -0.5)
        cmds.commit_and_wait()
        total = [0 if f else t for t, f in zip(total, finished)]
        total = [t + n for t, n in zip(total, new)]
        assert kv.to_numpy().tolist() == total
        T, got = table.to_numpy().reshape(4, width), from_bits(out.to_numpy(), dtype).reshape(cap, -1, dim)
        assert count3.to_numpy()[0] == n_blocks - sum(-(-t // bs) for t in total)
        live = np.concatenate([T[s, :-(-t // bs)] for s, t in enumerate(total)])
        assert len(set(live.tolist())) == len(live)
        at = 0
        for s, (t, n) in enumerate(zip(total, new)):
            if n == 0:
                continue
            j = np.arange(t)
            rows = [device.alloc_buffer(t * heads * dim, dtype) for _ in range(2)]
            kkv.kv_gather(cmds, cache, up(T[s][j // bs] * bs + j % bs), t, *rows)
            cmds.commit_and_wait()
            K, V = (from_bits(r.to_numpy(), dtype).astype(np.float64).reshape(t, heads, dim) for r in rows)
            x = from_bits(q[at:at + n], dtype).astype(np.float64)
            for h in range(heads * group):
                z = x[:, h] @ K[:, h // group].T * dim ** -0.5
                z[np.arange(t)[None, :] > np.arange(t - n, t)[:, None]] = -np.inf
                p = np.exp(z - z.max(1, keepdims=True))
                want = (p / p.sum(1, keepdims=True)) @ V[:, h // group]
                # The gathered rows are rounded to T (2^-9 each), which the cache's values are not.
                size = (np.abs(x[:, h]) @ np.abs(K[:, h // group]).T * dim ** -0.5).max(1, keepdims=True)
                assert (np.abs(got[at:at + n, h] - want) <=
                        2.0 ** -7 * np.abs(want) + (2.0 ** -8 * size + 2.0 ** -7) * np.abs(V[:, h // group]).max()).all()
            at += n
        lens, count = kv, count3
