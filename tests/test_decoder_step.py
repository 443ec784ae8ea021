"""A decoder layer's steps with the operators between its products together:
places planned, queries and keys rotated on the way into the 4-bit cache,
attention with capped and falling scores and prefixes over it, the grouped
router, the routed experts' product and their combination, against float64 over
what each step hands on.
"""
import numpy as np
import pytest

from cider_press_amd.kernels import gather as kgather
from cider_press_amd.kernels import kv as kkv
from cider_press_amd.kernels import moe as kmoe
from cider_press_amd.synthetic import from_bits, make_weight, to_bits
from test_kv_cache import NONE, _rows
from test_kv_rotary import frequencies_of, rotate
from test_kv_scores import make, standard_slopes
from test_moe_grouped import route

pytestmark = pytest.mark.gpu
DTYPE, DIM, GS, BS, KV_HEADS, GROUP, WIDTH, BLOCKS = "bf16", 64, 32, 16, 2, 4, 8, 24
EXPERTS, TOP_K, N = 32, 4, 64
HEADS, HIDDEN = KV_HEADS * GROUP, KV_HEADS * GROUP * DIM


def attend(q, k, v, positions, prefix, cap, slopes):
    """float64: q [n, heads, dim], k, v [t, kv heads, dim]."""
    out, j = np.zeros(q.shape), np.arange(len(k))[None, :]
    seen = (j <= positions[:, None]) | (j < prefix)
    for h in range(HEADS):
        z = cap * np.tanh(q[:, h] @ k[:, h // GROUP].T * DIM ** -0.5 / cap) + slopes[h] * (j - positions[:, None])
        z = np.where(seen, z, -np.inf)
        p = np.exp(z - z.max(1, keepdims=True))
        out[:, h] = (p / p.sum(1, keepdims=True)) @ v[:, h // GROUP]
    return out


def test_steps(device, library, oracle):
    """Prompts, decoded tokens, a request that ends while another comes; every step also replayed from a graph."""
    rng = np.random.default_rng(11)
    up = lambda a: device.upload(np.asarray(a, np.uint32).reshape(-1), "u32")
    cache = kkv.KvCache(device, DTYPE, BLOCKS, BS, KV_HEADS, DIM, GS)
    table, free = up(np.full((4, WIDTH), NONE)), up(rng.permutation(BLOCKS))
    lens, count, prefix = up([0] * 4), up([BLOCKS]), [5, 0, 20, 3]
    frequencies, slopes, cap = frequencies_of(DIM), standard_slopes(HEADS), 6.0
    F, S, P = device.upload(frequencies, "f32"), device.upload(slopes, "f32"), up(prefix)
    weights = [make_weight(rng, N, HIDDEN, 64, 4, DTYPE) for _ in range(EXPERTS)]
    w_q, s, b = (np.concatenate([w[i] for w in weights]) for i in range(3))
    W, SC, B = device.upload(w_q.reshape(-1), "u32"), device.upload(s.reshape(-1), DTYPE), device.upload(b.reshape(-1), DTYPE)
    bias = (rng.standard_normal(EXPERTS) * 0.05).astype(np.float32)
    BIAS = device.upload(bias, "f32")
    cmds = device.commands()
    total = [0] * 4
    steps = [([30, 16, 1, 0], [0] * 4), ([1, 1, 40, 0], [0] * 4), ([1, 0, 1, 45], [0, 1, 0, 0]), ([1, 5, 1, 1], [0] * 4)]
    for new, finished in steps:
        n = sum(new)
        cap_rows = n + 2  # two tokens of padding
        lens2, count2, starts, kv, slots, pos, left = (device.alloc_buffer(k, "u32") for k in
                                                       (4, 1, 5, 4, cap_rows, cap_rows, 1))
        fused = _rows(rng, cap_rows, HEADS + 2 * KV_HEADS, DIM, DTYPE)[0]
        X = device.upload(fused.reshape(-1), DTYPE)
        Q, A = (device.upload(np.full(cap_rows * HIDDEN, 0x5A5A, np.uint16), DTYPE) for _ in range(2))
        strides, k_at, v_at = ((HEADS + 2 * KV_HEADS) * DIM, DIM), HEADS * DIM, (HEADS + KV_HEADS) * DIM
        kkv.kv_release(cmds, up(finished), lens, table, WIDTH, BS, free, count, lens2, count2)
        kkv.kv_plan(cmds, lens2, up(new), table, WIDTH, BS, free, count2, starts, kv, slots, pos, left)
        logits = rng.standard_normal((n, EXPERTS)).astype(np.float32)
        L, rows = device.upload(logits.reshape(-1), "f32"), n * TOP_K
        experts, scores, lhs, rhs, inv = (device.alloc_buffer(rows, t) for t in ("u32", "f32", "u32", "u32", "u32"))
        offsets, Y, O = device.alloc_buffer(EXPERTS + 1, "u32"), device.alloc_buffer(rows * N, DTYPE), \
            device.alloc_buffer(n * N, DTYPE)

        def layer():
            kkv.kv_append_rotary(cmds, cache, X, X.slice(k_at, len(X) - k_at), X.slice(v_at, len(X) - v_at), slots, pos, F,
                                 Q, cap_rows, HEADS, q_strides=strides, k_strides=strides, v_strides=strides)
            kkv.kv_attention_scored(cmds, cache, Q, table, WIDTH, starts, kv, A, cap_rows, HEADS, 4, max(new), WIDTH * BS,
                                    DIM ** -0.5, softcap=cap, slopes=S, prefix_lens=P)
            kmoe.moe_route_grouped(cmds, L, n, EXPERTS, TOP_K, True, experts, scores, lhs, rhs, inv, offsets, sigmoid=True,
                                   bias=BIAS, n_groups=4, top_groups=2, group_best=2, scale=2.5)
            kgather.affine_gather_qmm(cmds, library, A, W, SC, B, lhs, rhs, Y, rows, N, HIDDEN, EXPERTS, 64, 4,
                                      sorted_indices=True, x_rows=n)
            kmoe.moe_combine(cmds, Y, scores, inv, n, TOP_K, N, O)

        layer()
        cmds.commit_and_wait()
        first = [x.to_numpy() for x in (Q, A, experts, scores, O)]
        cmds.begin_capture()
        layer()
        graph = cmds.end_capture()
        for _ in range(2):  # the same tokens into the same slots again
            for x in (Q, A):
                x.write(np.full(len(x), 0x5A5A, np.uint16))
            graph.launch(cmds)
            cmds.commit_and_wait()
            for x, y in zip((Q, A, experts, scores, O), first):
                assert np.array_equal(x.to_numpy(), y)
        total = [(0 if f else t) + m for t, f, m in zip(total, finished, new)]
        assert kv.to_numpy().tolist() == total
        positions = pos.to_numpy()
        want_q = rotate(fused[:, :HEADS], DTYPE, positions, frequencies)
        got_q, got_a = (x.reshape(cap_rows, HEADS, DIM) for x in first[:2])
        assert np.array_equal(got_q[:n], want_q[:n]) and (got_q[n:] == 0x5A5A).all() and (got_a[n:] == 0x5A5A).all()
        T, at = table.to_numpy().reshape(4, WIDTH), 0
        for r, (t, m) in enumerate(zip(total, new)):
            if m == 0:
                continue
            j = np.arange(t)
            outs = [device.alloc_buffer(t * KV_HEADS * DIM, DTYPE) for _ in range(2)]
            kkv.kv_gather(cmds, cache, up(T[r][j // BS] * BS + j % BS), t, *outs)
            cmds.commit_and_wait()
            K, V = (from_bits(x.to_numpy(), DTYPE).astype(np.float64).reshape(t, KV_HEADS, DIM) for x in outs)
            q = from_bits(want_q[at:at + m], DTYPE).astype(np.float64)
            assert positions[at:at + m].tolist() == list(range(t - m, t))
            want = attend(q, K, V, np.arange(t - m, t), prefix[r], cap, slopes)
            got = from_bits(got_a[at:at + m], DTYPE).astype(np.float64)
            # The gathered rows are rounded to T (2^-8 each), which the cache's values are not; scores through a cap of
            # slope 1 at most.
            for h in range(HEADS):
                size = (np.abs(q[:, h]) @ np.abs(K[:, h // GROUP]).T * DIM ** -0.5).max(1, keepdims=True)
                assert (np.abs(got[:, h] - want[:, h]) <= 2.0 ** -7 * np.abs(want[:, h]) +
                        (2.0 ** -8 * size + 2.0 ** -7) * np.abs(V[:, h // GROUP]).max()).all()
            at += m
        picks, weight = route(logits, TOP_K, sigmoid=True, bias=bias, n_groups=4, top_groups=2, group_best=2, scale=2.5)
        assert np.array_equal(first[2].reshape(n, TOP_K), picks)
        dense = oracle.gather_qmm_ref(first[1][:n * HIDDEN].reshape(n, HIDDEN), np.repeat(np.arange(n, dtype=np.uint32), TOP_K),
                                      picks.reshape(-1), w_q, s, b, rows, N, HIDDEN, 64, 4, DTYPE).reshape(n, TOP_K, N)
        dense = from_bits(to_bits(dense.astype(np.float32), DTYPE), DTYPE).astype(np.float64)
        want = (weight[:, :, None] * dense).sum(1)
        got = from_bits(first[4], DTYPE).astype(np.float64).reshape(n, N)
        # Each expert's row is rounded to T, on either side from sums in another order (one unit), then the sum is.
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -7 * (weight[:, :, None] * np.abs(dense)).sum(1)).all()
        lens, count = kv, left


def test_graphs_of_one_session(device):
    """Graphs that share a session's scratch (arrival counters, histograms, parts of split keys), replayed in turn."""
    rng = np.random.default_rng(6)
    cmds = device.commands()
    few, many, b = _router(device, rng, cmds, 20), _router(device, rng, cmds, 300), make(
        rng, device, (DTYPE, DIM, GS, BS, KV_HEADS, GROUP), [1, 1], [900, 4000], cap=6.0, slopes=True)
    want = b.run(cmds=cmds)
    b.check(want)
    graphs = []
    for encode in (few[0], lambda: b.encode(cmds), many[0]):
        cmds.begin_capture()
        encode()
        graphs.append(cmds.end_capture())
    for _ in range(3):
        for _, out, _ in (few, many):
            out.write(np.zeros(len(out), np.uint32))
        b.keep[5].write(np.zeros(len(b.keep[5]), np.uint16))
        for graph in graphs + graphs[::-1]:
            graph.launch(cmds)
        cmds.wait()
        for _, out, picks in (few, many):
            assert np.array_equal(out.to_numpy(), picks)
        assert np.array_equal(b.keep[5].to_numpy().reshape(want.shape), want)
        few[0]()
        cmds.wait()
        assert np.array_equal(few[1].to_numpy(), few[2])


def _router(device, rng, cmds, tokens):
    """(encode, buffer of experts, what belongs there)"""
    logits = rng.standard_normal((tokens, EXPERTS)).astype(np.float32)
    L, rows = device.upload(logits.reshape(-1), "f32"), tokens * TOP_K
    out = [device.alloc_buffer(rows, t) for t in ("u32", "f32", "u32", "u32", "u32")] + \
        [device.alloc_buffer(EXPERTS + 1, "u32")]
    kw = dict(sigmoid=True, n_groups=4, top_groups=2, group_best=2)
    return (lambda: kmoe.moe_route_grouped(cmds, L, tokens, EXPERTS, TOP_K, True, *out, **kw), out[0],
            route(logits, TOP_K, **kw)[0].reshape(-1))
