"""Which kernel a product's size selects: that the tests of the large kernels reach them, every instance of them, and where the limits lie."""
import ctypes as C

import pytest

from ivae_amd import _lib
from tests import operator_shapes as S

GELU, LRELU = 4, 1


def test_sizes_of_the_large_tests_reach_the_large_kernels():
    for size in S.BOTH:
        for dt in (S.F32, S.BF16, S.F16):
            for act in (0, GELU, LRELU):
                for backward in (0, 1):
                    assert S.plan(*size, dt, act, backward)[0] == S.LARGE, (size, dt, act, backward)


@pytest.mark.parametrize("dt", [S.F32, S.BF16, S.F16])
def test_sizes_of_the_large_tests_reach_every_instance(dt):
    """Every tile, number of buffers, and sums whole and split, in both directions."""
    forward = {S.instance(S.plan(*s, dt, act, 0), dt)[:3] for s in S.BOTH for act in (0, GELU)}
    tiles = [(256, None), (128, None)] if dt == S.F32 else [(256, None), (128, True), (128, False)]
    assert {f[:2] for f in forward} == set(tiles) and {f[2] for f in forward} == {False, True}
    for act in (0, GELU):
        back = {S.instance(S.plan(*s, dt, act, 1), dt) for s in S.BOTH}
        assert {b[:2] for b in back} == set(tiles), back
        assert {b[2] for b in back} == {b[3] for b in back} == {False, True}


def test_limits():
    """Few rows; a product's operations; rows that no 32-bit offset reaches; fp16 slopes whose gradients leave the range of a pair."""
    assert S.plan(64, 200, 200, S.F32)[0] == S.ROWS and S.plan(65, 200, 200, S.F32)[0] == S.TILES
    assert S.plan(32, 4096, 4096, S.F32)[0] == S.ROWS and S.plan(33, 4096, 4096, S.F32)[0] == S.TILES and S.plan(64, 4096, 4100, S.F32)[0] == S.ROWS
    assert S.plan(64, 4096, 4096, S.F16)[0] == S.ROWS and S.plan(65, 4096, 4096, S.F16)[0] == S.LARGE
    assert S.plan(1024, 1024, 1024, S.F16)[0] == S.LARGE and S.plan(1024, 1024, 1000, S.F16)[0] == S.TILES
    assert S.plan(4096, 4096, (1 << 21) + 8, S.F16)[0] == S.TILES
    for slope, kernel in ((16.0, S.LARGE), (-16.0, S.LARGE), (16.5, S.TILES), (float("inf"), S.TILES), (float("nan"), S.TILES)):
        assert S.plan(4096, 1024, 1024, S.F16, LRELU, 1, slope)[0] == kernel, slope
        assert S.plan(4096, 1024, 1024, S.BF16, LRELU, 1, slope)[0] == S.LARGE
        assert S.plan(4096, 1024, 1024, S.F16, 0, 1, 0.1)[0] == S.LARGE


def test_plan_refuses():
    L, out = _lib.lib(), (C.c_int32 * 5)()
    lin = _lib.IvaeLinear(4, 8, 8, 0, 0, .1, 8, 8, 8)
    assert L.ivae_debug_linear_plan(None, 0, out) == -3 and L.ivae_debug_linear_plan(lin, 0, None) == -3
    assert L.ivae_debug_linear_plan(_lib.IvaeLinear(4, 0, 8, 0, 0, .1, 8, 8, 8), 0, out) == -1
    assert L.ivae_debug_linear_plan(lin, 0, out) == 0 and out[0] == 0


def test_sizes_of_the_accuracy_tests():
    """Gradients of both kernels with an activation in the 16-bit types, and forward products of split fp32."""
    from tests import test_gpu_operators_accuracy as T
    for dt in (S.BF16, S.F16):
        for act in (LRELU, GELU):
            assert [S.plan(*s, dt, act, 1)[0] for s in T.SIZES] == [S.TILES, S.TILES, S.LARGE, S.LARGE]
    for s in ((1024, 2048, 1300), (1100, 1501, 1003), (4100, 520, 2003)):
        assert S.plan(*s, S.F32)[0] == S.LARGE
