"""Grouped routing of many tokens (kernels/moe.hip) whose workgroups have too few
rows each for histograms of their own, in a session of the default scratch.

No reference counterpart; semantics in include/cpq.h.
"""
import numpy as np
import pytest

from test_moe import np_sort
from test_moe_grouped import route, run


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k,groups,top,best", [
    (131072, 1024, 1, 1, 1, 1), (131072, 64, 1, 4, 2, 1), (66000, 33, 2, 3, 2, 2), (20001, 1000, 4, 10, 4, 2),
    (24001, 256, 8, 8, 4, 2), (24001, 256, 9, 8, 4, 2)])
def test_few_rows_a_workgroup(device, tokens, experts, k, groups, top, best):
    """On either side of where the routing workgroups' histograms are kept (8 and 9 picks).  The tokens repeat 300
    different ones, of which the definition's picks are taken."""
    rng = np.random.default_rng(tokens + k)
    rows, of = rng.standard_normal((300, experts)).astype(np.float32), rng.integers(0, 300, tokens)
    kw = dict(sigmoid=True, n_groups=groups, top_groups=top, group_best=best)
    _, (picks, scores, lhs, rhs, inv, offsets) = run(device, rows[of], "f32", k, **kw)
    want, weights = route(rows, k, **kw)
    assert np.array_equal(picks.reshape(tokens, k), want[of])
    np.testing.assert_allclose(scores.reshape(tokens, k), weights[of], rtol=2.0 ** -24 * 1.001, atol=2.0 ** -149)
    for got, ref in zip((lhs, rhs, inv, offsets), np_sort(picks, k, experts)):
        assert np.array_equal(got, ref)
