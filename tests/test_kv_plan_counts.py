"""What kv_plan reports of tokens without a place, past 32 bits (test_kv_cache.py:
run_plan)."""
import numpy as np
import pytest

from test_kv_cache import NONE, run_plan


@pytest.mark.gpu
@pytest.mark.parametrize("new,count", [([0xFFFFFFFF, 5], "1 * 2^32 token(s)"), ([0xFFFFFFFF, 0xFFFFFFFF, 6], "2 * 2^32 token(s)"),
                                       ([0xFFFFFFFF, 0xFFFFFFFF, 12], "2 * 2^32 + 6 token(s)"),
                                       ([0xFFFFFFFF, 4], "kv_plan: 4294967295 token(s)"), ([4, 1], "kv_plan: 1 token(s)")])
def test_counts_past_32_bits(device, new, count):
    """A total that is a multiple of 2^32 is an error as any other."""
    table = np.full((len(new), 4), NONE, np.uint32)
    got, message = run_plan(device, [0] * len(new), new, table, 16, np.arange(9), 9, 4)
    assert count in message
    assert np.array_equal(got[1], [4] + [0] * (len(new) - 1)) and got[5] == 8
