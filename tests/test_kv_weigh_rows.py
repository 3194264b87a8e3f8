"""CPU checks of the attention weights' kernels of many rows: which rows see a block of positions, and which workgroups and
workspace a batch gets."""
import ctypes as C

import numpy as np
import pytest

import aoship

I = C.c_int


def _visible(g, window, count, length, k0, k1):
    f = aoship.lib().aoship_internal_kv_weigh_rows
    f.restype, f.argtypes = None, [I] * 6 + [C.c_void_p]
    out = (I * 2)()
    f(g, window, count, length, k0, k1, out)
    return out[0], out[1]


@pytest.mark.parametrize("g", [1, 3, 7, 40])
@pytest.mark.parametrize("window", [0, 1, 9, 100])
def test_rows_that_see_a_block(g, window):
    """Against the definition: the first and the last row that see some of a block, with padding in front too"""
    rng = np.random.default_rng(g + window)
    for _ in range(300):
        count, length = int(rng.integers(1, 60)), int(rng.integers(1, 200))
        k0 = int(rng.integers(0, length))
        k1 = int(min(length, k0 + rng.integers(1, 65)))
        p = length - count + np.arange(count)
        sees = (p >= k0) & ((p - window + 1 <= k1 - 1) if window else True)
        ra, rb = _visible(g, window, count, length, k0, k1)
        t = np.flatnonzero(sees)
        if len(t):
            assert (ra, rb) == (t[0] * g, (t[-1] + 1) * g)
        else:
            assert ra >= rb


@pytest.mark.parametrize("length", [1 << 28, 306783379, (1 << 29) + 5, (1 << 30) - 1, 1 << 30])
@pytest.mark.parametrize("g", [2, 3, 4, 7, 16, 40])
def test_rows_of_a_block_far_before_the_window(g, length):
    """A row's distance to a block, times the heads of a group, passes 2^31: no row sees it"""
    for count in (1, 20, 1000):
        for k0 in (0, 256, 1 << 20, length // 4 // 256 * 256):
            ra, rb = _visible(g, 4096, count, length, k0, k0 + 256)
            assert ra >= rb and rb <= 0, (count, k0, ra, rb)
        last = (length - 1) // 256 * 256
        assert _visible(g, 4096, count, length, last, length) == (max(0, last - (length - count)) * g, count * g)
