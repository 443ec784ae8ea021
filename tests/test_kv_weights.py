"""Attention over the key/value cache: weights far below the largest keep their
precision (test_kv_cache.py: Batch)."""
import numpy as np
import pytest

from cider_press_amd.synthetic import from_bits, to_bits
from test_kv_cache import Batch, dequantize, quantize


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q", [1, 5, 60])
@pytest.mark.parametrize("size", [1.0, 1.5, 1.9296875, 2.1875, 2.25])
def test_small_weights_beside_sinks(device, dtype, q, size):
    """Every 32nd key takes nearly all of a row's weight and has zeros for values;
    the others weigh w = 2^-11.5 to 2^-26 of it and make the output.  A weight is
    off by half a unit of f16, 2^-11 of itself, and 2^-35 of the row's largest, values
    by 2^-11, the output by half a unit of T; keys and queries are exact here."""
    rng = np.random.default_rng(int(size * 64) + q)
    n = 700
    b = Batch(rng, device, dtype, 64, 32, 16, 1, 4, [q], [n])
    sink = np.arange(n) % 32 == 0
    k = np.where(sink[:, None, None], size, 0.0) * np.ones((n, 1, 64))
    v = np.where(sink[:, None, None], 0.0, 1.0 + 0.5 * rng.random((n, 1, 64)))
    parts = [quantize(from_bits(to_bits(x.astype(np.float32), dtype), dtype).astype(np.float32), 32, dtype) for x in (k, v)]
    b.host.put(b.table[0][np.arange(n) // 16] * 16 + np.arange(n) % 16, *parts)
    b.k[0], b.v[0] = (dequantize(*p, 32, dtype) for p in parts)
    b.q_bits = to_bits(np.ones(b.q.shape, np.float32), dtype)
    b.q = np.ones(b.q.shape)
    want, _ = b.expect(scale=0.125)
    got = from_bits(b.run(scale=0.125), dtype).astype(np.float64)
    w = np.exp(-8.0 * size)  # 64 dimensions of 1 x size, scale 1/8
    unit = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0  # subnormal outputs
    limit = 1.02 * (unit + 2.0 ** -10 + 2.0 ** -35 / w) * np.abs(want) + tiny
    assert (np.abs(got - want) <= limit).all(), (np.abs(got - want) / np.abs(want)).max()


@pytest.mark.gpu
@pytest.mark.parametrize("q", [1, 40])
def test_largest_scales(device, q):
    """Scales up to the largest accepted, whose product with log2(e) no float holds:
    the logits are ordinary."""
    rng = np.random.default_rng(q)
    n = 200
    b = Batch(rng, device, "bf16", 64, 32, 16, 1, 2, [q], [n], sharp=1e-33)
    x = from_bits(to_bits((rng.standard_normal((n, 1, 64)) * 1e-6).astype(np.float32), "bf16"), "bf16").astype(np.float32)
    v = from_bits(to_bits(rng.standard_normal((n, 1, 64)).astype(np.float32), "bf16"), "bf16").astype(np.float32)
    parts = [quantize(a, 32, "bf16") for a in (x, v)]
    b.host.put(b.table[0][np.arange(n) // 16] * 16 + np.arange(n) % 16, *parts)
    b.k[0], b.v[0] = (dequantize(*p, 32, "bf16") for p in parts)
    b.check(b.run(scale=3.3e38), scale=3.3e38)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,gs", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
@pytest.mark.parametrize("q,causal,window", [(1, True, 0), (130, True, 0), (70, False, 0), (200, True, 150)])
def test_f16_keeps_keys_and_weights(device, dim, gs, q, causal, window):
    """At T = f16 no more is lost than the output's rounding and the values' (a
    root mean square of 2.07e-4 of each, 2.9e-4 of both), for few rows and many."""
    rng = np.random.default_rng(dim + gs + q)
    b = Batch(rng, device, "f16", dim, gs, 16, 2, 4, [q, q + 1], [800, q + 1], sharp=2.0)
    want, _ = b.expect(causal, window)
    got = from_bits(b.run(causal, window), "f16").astype(np.float64)
    assert np.linalg.norm(got - want) <= 3.2e-4 * np.linalg.norm(want)
