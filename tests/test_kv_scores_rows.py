"""Attention for many rows (kernels/kv_attention.hpp) with scores that are capped,
biased or both: a row's result is its own, whatever the other queries and heads of
its wave look at.

No reference counterpart; semantics in include/cpq.h.
"""
import numpy as np
import pytest

from cider_press_amd.synthetic import from_bits, to_bits
from test_kv_scores import make

KINDS = [dict(), dict(cap=30.0), dict(cap=1024.0), dict(slopes=True), dict(cap=30.0, slopes=True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim,gs", [("bf16", 64, 64), ("bf16", 128, 64), ("f16", 128, 32), ("bf16", 256, 128)])
@pytest.mark.parametrize("kind", range(len(KINDS)))
def test_rows_are_their_own(device, dtype, dim, gs, kind):
    """One query looks sharply, so that its weights leave f16's range where the others' do not, or sees hardly any
    difference: no bit of the other rows changes."""
    b = make(np.random.default_rng(dim + kind), device, (dtype, dim, gs, 16, 2, 4), [72], [700], **KINDS[kind], sharp=2.0)
    want = b.run()
    b.check(want)
    q = from_bits(b.q_bits, dtype)
    for row, factor in ((3, 12.0), (3, 0.0), (40, 12.0), (71, -5.0)):
        x = q.copy()
        x[row] *= factor
        b.q_bits = to_bits(x, dtype)
        got = b.run()
        assert not np.array_equal(got[row], want[row])
        others = np.arange(72) != row
        apart = got[others] != want[others]
        assert not apart.any(), f"{apart.sum()} values of other rows with query {row} times {factor}"
