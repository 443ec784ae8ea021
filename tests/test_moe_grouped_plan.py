"""How the grouped router divides tokens over workgroups (kernels/moe.hip), seen by
the histograms that it keeps in session scratch."""
import ctypes

from cider_press_amd import _lib
from cider_press_amd.kernels import moe as kmoe


def scratch_bytes(tokens, experts, cus):
    f = _lib.lib()._ZN3cpq25moe_grouped_scratch_bytesEiiRK14cpq_moe_routeri  # internal: no C name
    f.restype, f.argtypes = ctypes.c_size_t, [ctypes.c_int, ctypes.c_int, ctypes.c_char_p, ctypes.c_int]
    return f(tokens, experts, kmoe._router(True, None, 1, 1, 1, True, 1.0), cus)


def test_compute_units():
    """Four tokens a workgroup while every compute unit of this device has at most one, then eight, then 16."""
    for cus in (32, 64, 128, 256, 304):
        for tokens, per in ((1, 4), (4 * cus, 4), (4 * cus + 1, 8), (8 * cus, 8), (8 * cus + 1, 16), (16 * cus + 5, 16)):
            assert scratch_bytes(tokens, 64, cus) == -(-tokens // per) * 64
    assert scratch_bytes(1000, 256, 256) == 250 * 256 and scratch_bytes(1000, 256, 128) == 125 * 256
