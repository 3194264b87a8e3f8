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


def _shape(nkv, nh, n, T, new, L):
    f = aoship.lib().aoship_internal_kv_weigh_shape
    f.restype, f.argtypes = C.c_size_t, [I] * 6 + [C.c_void_p]
    out = (I * 7)()
    size = f(nkv, nh, n, T, new, L, out)
    return size, dict(zip(("few", "rc", "each", "chunks", "piece_each", "pieces", "lpad"), out))


def _documented(nkv, nh, n, T, L):
    """the header's bytes of a batch whose sequences may have more than 32 rows"""
    blocks = -(-L // 256)
    return 8 * T * nh * (blocks + 1) + nkv * 256 * blocks * (4 * (T * nh // nkv / 256) + 5 * n) + 4 * 2 ** 20 + 4096


@pytest.mark.parametrize("nkv,nh,decodes,prompt,L", [(4, 28, 255, 8192, 32768), (4, 28, 63, 4001, 16000),
                                                     (8, 40, 255, 8192, 131072), (2, 14, 1023, 300, 9000), (8, 24, 7, 300, 900)])
def test_one_prompt_beside_single_tokens(nkv, nh, decodes, prompt, L):
    """The launches and the workspace follow the batch's rows, not its sequences times the longest one's"""
    n, T = decodes + 1, decodes + prompt
    size, d = _shape(nkv, nh, n, T, prompt, L)
    assert 0 < size <= _documented(nkv, nh, n, T, L)
    g = nh // nkv
    assert d["each"] == 0 and d["chunks"] <= T * g // d["rc"] + n and d["pieces"] <= T * g // 256 + n
    most = aoship.lib().aoship_internal_kv_weigh_most
    most.restype, most.argtypes = C.c_size_t, [I] * 6
    assert most(nkv, nh, n, T, prompt, L) >= size


@pytest.mark.parametrize("seed", range(20))
def test_shares_hold_every_row(seed):
    """Random batches: each sequence's shares are its own, enough for its rows, and within the launch and the workspace."""
    rng = np.random.default_rng(seed)
    base = aoship.lib().aoship_internal_kv_weigh_share
    base.restype, base.argtypes = C.c_longlong, [I] * 5
    for _ in range(60):
        n, top = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 11))
        new = np.where(rng.random(n) < rng.random(), 1, rng.integers(0, top + 1, n))
        skip, L = int(rng.integers(0, 3) * rng.integers(0, 5)), int(2 ** rng.uniform(0, 15))
        starts = skip + np.concatenate([[0], np.cumsum(new)])
        T, most = int(starts[-1] + rng.integers(0, 2) * rng.integers(0, 300)), max(1, int(new.max()))
        if T == 0:
            continue
        nkv = int(rng.choice([1, 2, 8]))
        g = int(rng.choice([1, 3, 7, 40]))
        size, d = _shape(nkv, nkv * g, n, T, most, L)
        assert size > 0
        if d["few"]:
            assert most * g <= 32
            continue
        assert size <= _documented(nkv, nkv * g, n, T, L)
        # the parts: chunks' weights, maxima and sums of blocks, of rows
        assert 4 * d["chunks"] * nkv * d["lpad"] + 8 * T * nkv * g * (d["lpad"] // 256 + 1) <= size
        for unit, each, count in ((d["rc"], d["each"], d["chunks"]), (256, d["piece_each"], d["pieces"])):
            b = [base(unit, each, g, s, int(starts[s])) for s in range(n)] + [count]
            for s in range(n):
                assert b[s + 1] - b[s] >= -(-int(new[s]) * g // unit) and b[s] >= 0
            assert count == (n * each if each else T * g // unit + n) and each in (0, -(-most * g // unit))
        assert (d["each"] == 0) == (n * -(-most * g // 64) > 2 * (T * g // 64 + n))
