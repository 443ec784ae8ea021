"""Grouped routing of experts (kernels/moe.hip) against its definition in numpy
float64, token by token; the sort against a stable argsort.

No reference counterpart (its docs name the router as unbuilt); semantics in
include/cpq.h.
"""
import numpy as np
import pytest

from cider_press_amd import _lib
from cider_press_amd.kernels import Buffer
from cider_press_amd.kernels import moe as kmoe
from cider_press_amd.synthetic import from_bits, to_bits
from test_moe import np_sort


def route(logits, k, normalize=True, sigmoid=False, bias=None, n_groups=1, top_groups=1, group_best=1, scale=1.0):
    """Picks and scores [tokens, k], by the definition."""
    x = logits.astype(np.float64)
    picks, scores = [], []
    with np.errstate(all="ignore"):
        for row in x:
            if sigmoid:
                s = 1.0 / (1.0 + np.exp(-row))
            else:
                s = np.exp(row - np.fmax.reduce(row))
                s = s / s.sum()
            c = s if bias is None else s + bias.astype(np.float64)
            c = np.where(np.isnan(c), -np.inf, c)  # (no test has an infinite bias below beside a NaN)
            among = np.arange(len(c))
            if n_groups > 1:
                g = np.sort(c.reshape(n_groups, -1), 1)[:, ::-1][:, :group_best].sum(1)
                kept = sorted(range(n_groups), key=lambda i: (-g[i], i))[:top_groups]
                among = among[np.isin(among * n_groups // len(c), kept)]
            pick = sorted(among.tolist(), key=lambda e: (-c[e], e))[:k]
            w = s[pick]
            if normalize:
                w = np.zeros(k) if w.sum() == 0 else w / w.sum()
            picks.append(pick)
            scores.append(w * scale)
    return np.asarray(picks, np.uint32), np.asarray(scores)


def _buffers(device, rows, experts):
    return [device.upload(np.full(max(rows, 1), 77, np.uint32 if t == "u32" else np.float32), t)
            for t in ("u32", "f32", "u32", "u32", "u32")] + [device.alloc_buffer(experts + 1, "u32")]


def run(device, logits, dtype, k, normalize=True, bias=None, cmds=None, **kw):
    tokens, experts = logits.shape
    bits = logits.astype(np.float32) if dtype == "f32" else to_bits(logits.astype(np.float32), dtype)
    out = _buffers(device, tokens * k, experts)
    cmds = cmds or device.commands()
    kmoe.moe_route_grouped(cmds, device.upload(bits.reshape(-1), dtype), tokens, experts, k, normalize, *out,
                           bias=None if bias is None else device.upload(bias, "f32"), **kw)
    cmds.commit_and_wait()
    seen = bits if dtype == "f32" else from_bits(bits, dtype)
    return seen, [b.to_numpy()[:tokens * k] for b in out[:5]] + [out[5].to_numpy()]


def alike(x, sigmoid, bias, n_groups, top_groups):
    """Tokens whose last kept group and first left group have sums of two that are the same but for roundings.  (s_a + b_1)
    + (s_c + b_2) and (s_a + b_2) + (s_c + b_1) are one number; in fp64, with scores below 1, either is off from it by
    2^-53 for each s (an exponential's last bit) and each of three sums: 2^-51 in all, so their order is rounding's."""
    s = x.astype(np.float64)
    s = 1 / (1 + np.exp(-s)) if sigmoid else np.exp(s - s.max(1, keepdims=True))
    s = s if sigmoid else s / s.sum(1, keepdims=True)
    g = np.sort((s + bias.astype(np.float64)).reshape(len(x), n_groups, -1), 2)[..., -2:].sum(2)
    g = np.sort(g, 1)[:, ::-1]
    return g[:, top_groups - 1] - g[:, top_groups] <= 2.0 ** -51


def check(device, logits, dtype, k, either=None, **kw):
    """either: says of which tokens the kept groups are not determined."""
    seen, (experts, scores, lhs, rhs, inv, offsets) = run(device, logits, dtype, k, **kw)
    picks, want = route(seen, k, **kw)
    n = len(seen)
    sure = np.ones(n, bool) if either is None else ~either(seen)
    assert sure.mean() > 0.5
    assert np.array_equal(experts.reshape(n, k)[sure], picks[sure])
    # One rounding to fp32; exponentials and sums in fp64 are off by 2^-50.
    np.testing.assert_allclose(scores.reshape(n, k)[sure], want[sure], rtol=2.0 ** -24 * 1.001, atol=2.0 ** -149)
    for got, ref in zip((lhs, rhs, inv, offsets), np_sort(experts, k, logits.shape[1])):
        assert np.array_equal(got, ref)


def test_refusals():
    check_args = _lib.lib().cpq_check_moe_route_grouped_args

    def args(dtype="f32", tokens=5, experts=64, k=8, sigmoid=1, bias=None, groups=8, top=4, best=2, scale=1.0):
        b = None if bias is None else Buffer(None, bias, 64, "f32", 256)
        if b is not None:
            b._owner = b  # no memory of its own
        return check_args(_lib.DTYPES[dtype], tokens, experts, k,
                          kmoe._router(sigmoid, b, groups, top, best, True, scale))

    for good in (dict(), dict(tokens=0), dict(groups=1, top=1), dict(groups=64, top=8, best=1), dict(groups=64, top=64, best=1),
                 dict(bias=4096), dict(scale=-2.0), dict(k=16, top=2), dict(experts=1024, groups=64), dict(dtype="bf16")):
        assert args(**good) == _lib.OK, (good, _lib.last_error())
    for bad in (dict(dtype="u32"), dict(experts=0), dict(experts=1025), dict(k=0), dict(k=17), dict(experts=4, groups=1, top=1, k=5),
                dict(groups=0), dict(groups=7), dict(groups=65, experts=650), dict(top=0), dict(top=9), dict(best=0),
                dict(best=3), dict(groups=64, top=64, best=2), dict(k=9, top=1), dict(bias=4098),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(tokens=2**28, k=8), dict(tokens=2**62),
                dict(tokens=2**25 + 1, k=1)):
        assert args(**bad) == _lib.INVALID_ARGUMENT, bad
    assert check_args(0, 5, 64, 8, None) == _lib.INVALID_ARGUMENT
    assert _lib.lib().cpq_moe_route_grouped(None, 0, None, 0, 4, 1, None, *[None] * 6) == _lib.INVALID_ARGUMENT
    assert kmoe._ROUTER.size % 8 == 0


def test_buffer_checks():
    b = lambda n, t: Buffer(None, None, n, t, 4 * n)
    out = [b(8, "u32"), b(8, "f32"), b(8, "u32"), b(8, "u32"), b(8, "u32"), b(17, "u32")]
    go = lambda logits=b(64, "f32"), out=out, **kw: kmoe.moe_route_grouped(None, logits, 4, 16, 2, True, *out, **kw)
    for error, kw in ((TypeError, dict(bias=b(16, "bf16"))), (_lib.InvalidArgument, dict(bias=b(15, "f32"))),
                      (_lib.InvalidArgument, dict(logits=b(63, "f32"))), (TypeError, dict(out=out[::-1])),
                      (_lib.InvalidArgument, dict(out=out[:5] + [b(16, "u32")])),
                      (_lib.InvalidArgument, dict(out=[b(7, "u32")] + out[1:])),
                      (_lib.InvalidArgument, dict(n_groups=-1))):
        with pytest.raises(error):
            go(**kw)


SHAPES = [  # tokens, experts, k, groups, top_groups, group_best
    (16, 256, 8, 8, 4, 2), (1, 256, 8, 8, 4, 2), (33, 160, 6, 8, 3, 1), (700, 60, 4, 1, 1, 1), (40, 1024, 16, 64, 5, 2),
    (5, 1000, 16, 50, 3, 2), (300, 12, 2, 6, 2, 2), (2100, 64, 8, 4, 4, 2), (31, 4, 4, 1, 1, 2), (1, 1, 1, 1, 1, 1),
    (90, 65, 5, 13, 2, 1), (64, 512, 1, 64, 1, 1), (32, 48, 12, 16, 4, 2), (77, 320, 10, 5, 2, 2), (50, 130, 3, 2, 1, 2),
    (45, 64, 3, 64, 3, 1), (40, 990, 16, 33, 4, 2), (20, 1000, 7, 10, 3, 2), (100, 320, 13, 16, 8, 2), (37, 208, 9, 16, 5, 1),
    (60, 1023, 5, 3, 2, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("sigmoid,biased,normalize,scale", [(True, True, True, 2.5), (False, False, False, 16.0),
                                                            (False, True, True, 1.0), (True, False, False, -1.0)])
def test_route(device, shape, sigmoid, biased, normalize, scale):
    tokens, experts, k, groups, top, best = shape
    rng = np.random.default_rng(experts * 3 + k + sigmoid)
    logits = rng.standard_normal((tokens, experts)) * 2.0 - 0.5
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32) if biased else None
    for dtype in ("f32", "bf16", "f16"):
        check(device, logits, dtype, k, normalize=normalize, sigmoid=sigmoid, bias=bias, n_groups=groups, top_groups=top,
              group_best=best, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k,groups,top,best", [
    (8192, 256, 8, 8, 4, 2), (8193, 256, 3, 8, 4, 2), (2560, 1024, 8, 8, 2, 2), (2561, 1024, 8, 8, 2, 2), (65535, 32, 1, 4, 1, 1), (65536, 32, 1, 4, 1, 1), (70001, 2, 2, 2, 2, 1),
    (2100, 1024, 5, 1, 1, 1), (1100, 1000, 16, 10, 4, 2), (40000, 17, 3, 1, 1, 1), (65535, 1, 1, 1, 1, 1)])
def test_many_tokens(device, tokens, experts, k, groups, top, best):
    """On either side of where the sort scans its histograms; all tokens with one expert, too."""
    rng = np.random.default_rng(tokens)
    logits = rng.standard_normal((tokens, experts)).astype(np.float32)
    kw = dict(sigmoid=True, n_groups=groups, top_groups=top, group_best=best)
    check(device, logits, "f32", k, **kw)
    rows = rng.permutation(tokens)[:300]
    logits[:] = np.linspace(3.0, -3.0, experts)  # the same picks for all but a few
    logits[rows] = logits[rows, ::-1]
    check(device, logits, "f32", k, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 50])
@pytest.mark.parametrize("sigmoid", [True, False])
def test_ties(device, tokens, sigmoid):
    """Equal scores, groups and all: the lower index."""
    for experts, k, groups, top, best in ((64, 8, 8, 3, 2), (200, 9, 10, 4, 1), (256, 16, 1, 1, 1), (320, 7, 64, 2, 2)):
        logits = np.zeros((tokens, experts))
        logits[1, ::3] = 1.0
        logits[2] = np.arange(experts) % 2
        logits[2, -1] = 1.0
        kw = dict(sigmoid=sigmoid, n_groups=groups, top_groups=top, group_best=best)
        check(device, logits, "f32", k, **kw)
        check(device, logits, "bf16", k, bias=np.full(experts, -0.25, np.float32), **kw)


@pytest.mark.gpu
def test_near_scores(device):
    """Scores and sums that fp32 would round together or change places of."""
    rng = np.random.default_rng(4)
    tokens, experts = 400, 128
    base = rng.standard_normal((tokens, 1)).astype(np.float32)
    logits = base * (1 + rng.integers(-3, 4, (tokens, experts)).astype(np.float32) * np.float32(2.0 ** -23))
    bias = (rng.integers(-2, 3, experts) * 2.0 ** -26).astype(np.float32)
    for sigmoid in (True, False):
        for groups, top, best in ((1, 1, 1), (8, 4, 2)):
            check(device, logits, "f32", 8, sigmoid=sigmoid, n_groups=groups, top_groups=top, group_best=best)
            either = (lambda x: alike(x, sigmoid, bias, groups, top)) if groups > 1 else None
            check(device, logits, "f32", 8, either, sigmoid=sigmoid, bias=bias, n_groups=groups, top_groups=top,
                  group_best=best)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [6, 60])
def test_special_logits(device, tokens):
    """-Inf (experts masked out), far logits, all masked, NaN, +Inf: picks stay experts, each one once."""
    rng = np.random.default_rng(tokens)
    experts, k = 96, 6
    kw = dict(n_groups=8, top_groups=3, group_best=2)
    logits = rng.standard_normal((tokens, experts))
    logits[0, 5:90] = -np.inf
    logits[1] *= 1e4
    logits[2, ::2] = -800.0
    for sigmoid in (True, False):
        check(device, logits, "f32", k, sigmoid=sigmoid, **kw)
    dark = np.full((tokens, experts), -np.inf)
    check(device, dark, "f32", k, sigmoid=True, **kw)  # sums of 0
    logits[3, 7], logits[4], logits[5, 50] = np.nan, np.nan, np.inf
    check(device, logits, "f32", k, sigmoid=True, **kw)
    for bias in (None, np.where(np.arange(experts) % 3, 0, -np.inf).astype(np.float32)):
        for sigmoid in (True, False):
            _, (picks, scores, lhs, rhs, inv, offsets) = run(device, logits, "f32", k, sigmoid=sigmoid, bias=bias, **kw)
            picks = picks.reshape(tokens, k)
            assert picks.max() < experts and all(len(set(p)) == k for p in picks.tolist())
            assert sorted(inv.tolist()) == list(range(tokens * k)) and offsets[-1] == tokens * k
            if not sigmoid:
                assert np.isnan(scores.reshape(tokens, k)[3:6]).all()


@pytest.mark.gpu
def test_nothing_and_graph(device):
    rng = np.random.default_rng(2)
    _, got = run(device, np.zeros((0, 32)), "f32", 4, sigmoid=True, n_groups=4, top_groups=2)
    assert not got[5].any()
    for tokens in (8, 100):
        logits = rng.standard_normal((tokens, 128)).astype(np.float32)
        bias = device.upload(np.zeros(128, np.float32), "f32")
        L, out = device.upload(logits.reshape(-1), "f32"), _buffers(device, tokens * 8, 128)
        cmds = device.commands()
        encode = lambda: kmoe.moe_route_grouped(cmds, L, tokens, 128, 8, True, *out, sigmoid=True, bias=bias, n_groups=8,
                                                top_groups=4, group_best=2)
        cmds.begin_capture()
        encode()
        graph = cmds.end_capture()
        for i in range(3):
            logits = rng.standard_normal((tokens, 128)).astype(np.float32)
            b = (rng.standard_normal(128) * 0.1).astype(np.float32)
            L.write(logits.reshape(-1))
            bias.write(b)
            want, _ = route(logits, 8, sigmoid=True, bias=b, n_groups=8, top_groups=4, group_best=2)
            for go in (lambda: graph.launch(cmds), encode):
                out[0].write(np.zeros(tokens * 8, np.uint32))
                go()
                cmds.wait()
                assert np.array_equal(out[0].to_numpy().reshape(tokens, 8), want)
                assert np.array_equal(out[2].to_numpy(), np_sort(want.reshape(-1), 8, 128)[0])


@pytest.mark.gpu
def test_as_moe_route(device):
    """With nothing asked for it picks as moe_route does."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((70, 128)).astype(np.float32)
    _, got = run(device, logits, "f32", 8)
    out = _buffers(device, 560, 128)
    cmds = device.commands()
    kmoe.moe_route(cmds, device.upload(logits.reshape(-1), "f32"), 70, 128, 8, True, *out)
    cmds.commit_and_wait()
    for i in (0, 2, 3, 4, 5):
        assert np.array_equal(got[i], out[i].to_numpy())
    np.testing.assert_allclose(got[1], out[1].to_numpy(), rtol=2e-6)
