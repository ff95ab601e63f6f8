"""Which kernel a layer's call runs as: the sizes of the GPU tests reach all of them."""
import ctypes as C

from linear_plans import PLANS, UNREACHED, combinations


def test_the_sizes_reach_every_kernel():
    from frhot import _lib
    lib, plan = _lib.load(), (C.c_int32 * 4)()
    seen = set()
    for shape, way, splits, m, n, k in PLANS:
        assert lib.frhot_linear_debug_plan(n, k, m, way == "dma", 0, plan) == 0
        got = (plan[0], "gather" if plan[2] else "pack" if plan[3] else "dma", plan[1])
        assert got == (shape, way, splits), (m, n, k, got)
        seen.add((shape, way, splits > 1))
    assert seen == combinations() - UNREACHED


def test_refusals():
    from frhot import _lib
    lib, plan = _lib.load(), (C.c_int32 * 4)()
    for n, k, m in ((0, 8, 8), (8, 0, 8), (8, 8, 0), (65537, 8, 8), (8, 65537, 8), (8, 8, 2 ** 31)):
        assert lib.frhot_linear_debug_plan(n, k, m, 1, 0, plan) == -1
    assert lib.frhot_linear_debug_plan(8, 8, 8, 1, 0, None) == -1
