"""Sizes of products that the library's large kernels take, and the query that says so."""
import ctypes as C

from ivae_amd import _lib

F32, BF16, F16 = 0, 1, 2
ROWS, TILES, LARGE = 0, 1, 2        # few rows, 64 x 64 tiles, large tiles

# (rows, in, out); both directions of every type are the large kernels'
BOTH = [(2050, 1100, 1201), (4100, 520, 2003), (1100, 1501, 1003), (8200, 1032, 1100), (8192, 264, 4096), (1030, 4100, 4200), (520, 16384, 640),
        (4096, 4096, 4096), (300, 1100, 9000), (20000, 520, 264), (3000, 3000, 2990)]


def plan(m, k, n, dtype, act=0, backward=0, slope=.1):
    """(kernel, tile, parts of y or dx, parts of dw, blocks) of a call with dense tensors."""
    out = (C.c_int32 * 5)()
    rc = _lib.lib().ivae_debug_linear_plan(_lib.IvaeLinear(m, k, n, dtype, act, slope, k, n, n), backward, out)
    assert rc == 0, rc
    return tuple(out)


def instance(p, dtype):
    """What is a kernel of its own, and whether its sums are split: 16-bit tiles of 128 have four buffers up to 256 blocks, two beyond."""
    return (p[1], None if dtype == F32 or p[1] == 256 else p[4] <= 256, p[2] > 1, p[3] > 1)
