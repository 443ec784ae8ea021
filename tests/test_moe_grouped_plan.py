"""How the grouped router divides tokens over workgroups (kernels/moe.hip), seen by
the histograms that it keeps in session scratch."""
import ctypes

from cider_press_amd import _lib
from cider_press_amd.kernels import moe as kmoe


def scratch_bytes(tokens, experts, cus, top_k=1):
    f = _lib.lib()._ZN3cpq25moe_grouped_scratch_bytesEiiiRK14cpq_moe_routeri  # internal: no C name
    f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_int] * 3 + [ctypes.c_char_p, ctypes.c_int]
    return f(tokens, experts, top_k, kmoe._router(True, None, 1, 1, 1, True, 1.0), cus)


def test_compute_units():
    """Four tokens a workgroup while every compute unit of this device has at most one, then eight, then 16."""
    for cus in (32, 64, 128, 256, 304):
        for tokens, per in ((1, 4), (4 * cus, 4), (4 * cus + 1, 8), (8 * cus, 8), (8 * cus + 1, 16), (16 * cus + 5, 16)):
            assert scratch_bytes(tokens, 64, cus) == -(-tokens // per) * 64
    assert scratch_bytes(1000, 256, 256) == 250 * 256 and scratch_bytes(1000, 256, 128) == 125 * 256


def test_scratch():
    """Never past what the header says: 256 KiB, or 4 * n_experts bytes for every 128 rows."""
    for experts in (1, 2, 17, 64, 256, 600, 1000, 1024):
        for tokens in (1, 33, 1000, 5000, 8191, 65535, 65536, 131072, 1 << 22, 1 << 25):
            for top_k in {1, 2, 3, 8, 9, 16} & set(range(1, experts + 1)):
                most = max(256 * 1024, 4 * experts * -(-tokens * top_k // 128))
                assert scratch_bytes(tokens, experts, 256, top_k) <= most
    # One pick a token takes no more than moe_route does.
    assert scratch_bytes(131072, 1024, 256) == 131072 // 256 * 1024 * 4
