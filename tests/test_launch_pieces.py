"""CPU checks of calls whose workgroups pass what one grid may have: fewer than 2^32 threads."""
import ctypes as C

import aoship

I = C.c_int


def test_a_piece_is_a_grid():
    """Kernels have up to 1024 threads a workgroup (the eviction's choice); pieces are for all of them alike."""
    f = aoship.lib().aoship_internal_set_launch_most
    f.restype, f.argtypes = C.c_uint32, [C.c_uint32]
    most = f(5)
    assert f(0) == 5 and f(0) == most
    assert most * 1024 < 2 ** 32


def test_calls_that_one_grid_cannot_hold_are_accepted():
    """so that they have to be launched in pieces"""
    L = aoship.lib()
    shape = L.aoship_internal_kv_weigh_shape
    shape.restype, shape.argtypes = C.c_size_t, [I] * 6 + [C.c_void_p]
    out = (I * 7)()
    for nkv, nh, n, T, new, length in ((4, 8, 1, 1, 1, 1 << 30), (8, 40, 1 << 15, 1 << 18, 8, 1 << 14)):
        assert shape(nkv, nh, n, T, new, length, out) > 0
        assert not out[0] and out[3] * nkv * (out[6] // 256) * 256 >= 2 ** 32
    check = L.aoship_internal_logprobs_check
    check.restype, check.argtypes = I, [C.c_void_p, I, I, I, C.c_int64, C.c_void_p, C.c_void_p]
    o = aoship._LogProbsOut(entropy=4096)
    assert check(4096, 0, 1 << 26, 1, 1, None, C.byref(o)) == 0 and (1 << 26) * 256 >= 2 ** 32
    evict = L.aoship_internal_kv_evict_check
    evict.restype, evict.argtypes = I, [C.c_void_p, I, C.c_void_p, C.c_void_p]
    cfg, P, n, keep = aoship._KVConfig(1, 8, 64, 64, 1, 2), 4096, 1 << 15, 1 << 13
    b = aoship._KVBatch(n, 0, 0, keep, None, P, P, keep // 64)
    e = aoship._KVEvict(P, 8 * keep, keep, P, keep, 0, 0, P, keep // 64, P, 8 * keep, keep, None, 0, 0)
    assert evict(C.byref(cfg), 0, C.byref(b), C.byref(e)) == 0 and n * 8 * (keep // 64) * 256 >= 2 ** 32
