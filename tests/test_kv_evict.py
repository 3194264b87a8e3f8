"""CPU checks of rotary positions given to append, attention weights and eviction: what the calls refuse, with every bound on
both sides, and the workspace that a reservation covers."""
import ctypes as C

import numpy as np
import pytest

import aoship
from test_kv_cache import ALIGNED as P, CFG, _batch, _rows

I, V = C.c_int, C.c_void_p


def _fn(name, args, res=I):
    f = getattr(aoship.lib(), name)
    f.restype, f.argtypes = res, args
    return f


def _append_at(layer=0, batch=None, rows=None, rope=1, positions=P, stride=40):
    f = _fn("aoship_internal_kv_append_at_check", [V, I, I, V, V, V, C.c_int64])
    return f(C.byref(CFG), rope, layer, C.byref(batch or _batch()), C.byref(rows or _rows()), positions, stride)


def test_positions():
    assert _append_at() == 0  # (a table of one position: which are in it is seen on the device)
    assert _append_at(stride=0) == 0 and _append_at(stride=41) == 0
    for bad in (dict(stride=39), dict(stride=-40), dict(stride=1 << 40), dict(positions=None), dict(positions=P + 2),
                dict(rope=0), dict(rows=_rows(rotated=1)), dict(layer=2), dict(rows=_rows(k=None)),
                dict(batch=_batch(max_len=641)), dict(rows=_rows(num_heads=6))):
        assert _append_at(**bad) == -1, bad
        assert aoship.last_error().startswith("aoship_kv_append_at")
    assert _append_at(batch=_batch(n_tokens=0), positions=None) == 1


def _weigh(layer=0, batch=None, q=P, qs=1024, nh=8, scale=0.1, window=0, null=False, **kw):
    d = dict(prior=None, prior_seq=0, prior_head=0, out=P, out_seq=4 * 640, out_head=640)
    d.update(kw)
    f = _fn("aoship_internal_kv_weigh_check", [V, I, V, V, C.c_int64, I, C.c_float, I, V, C.POINTER(C.c_size_t)])
    w, n = aoship._KVWeights(**d), C.c_size_t()
    return f(C.byref(CFG), layer, C.byref(batch or _batch()), q, qs, nh, scale, window, None if null else C.byref(w), C.byref(n))


def test_weigh_accepts():
    assert _weigh() == 0 and _weigh(out=P + 4, out_seq=4 * 641, out_head=641) == 0
    assert _weigh(prior=2 * P, prior_seq=5000, prior_head=700) == 0
    assert _weigh(prior=P, prior_seq=4 * 640, prior_head=640) == 0  # in place
    assert _weigh(batch=_batch(n_seqs=1, n_tokens=1, max_new=1), out_seq=0) == 0
    assert _weigh(batch=_batch(n_tokens=0)) == 1 and _weigh(batch=_batch(max_len=0)) == 1


@pytest.mark.parametrize("kw", [dict(layer=2), dict(layer=-1), dict(q=None), dict(q=P + 8), dict(qs=1016), dict(qs=1028),
                                dict(nh=6), dict(nh=0), dict(nh=65540), dict(window=-1), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(scale=2.4e38), dict(null=True), dict(out=None), dict(out=P + 2),
                                dict(out_head=639), dict(out_seq=4 * 640 - 1), dict(out_head=1 << 40), dict(out_seq=1 << 40),
                                dict(prior=2 * P), dict(prior=P + 1, prior_seq=2560, prior_head=640),
                                dict(prior=P, prior_seq=2561, prior_head=640), dict(prior=P, prior_seq=4000, prior_head=700)],
                         ids=lambda k: "-".join(k))
def test_weigh_refuses(kw):
    assert _weigh(**kw) == -1
    assert aoship.last_error().startswith("aoship_kv_weigh")


def test_weigh_counts_its_work():
    big = dict(max_len=1 << 30, page_stride=1 << 24)
    wide = dict(out_seq=4 << 30, out_head=1 << 30)
    assert _weigh(batch=_batch(n_seqs=1, n_tokens=1, max_new=1, **big), **wide) == 0
    assert _weigh(batch=_batch(n_seqs=1, n_tokens=1 << 20, max_new=1 << 20, **big), **wide) == -1
    assert "too large" in aoship.last_error()


@pytest.mark.parametrize("seed", range(30))
def test_a_reservation_covers_smaller_batches(seed):
    rng = np.random.default_rng(seed)
    need = _fn("aoship_internal_kv_weigh_check", [V, I, V, V, C.c_int64, I, C.c_float, I, V, C.POINTER(C.c_size_t)])
    most = _fn("aoship_internal_kv_weigh_most", [I] * 6, C.c_size_t)
    for _ in range(200):
        nkv = int(rng.choice([1, 2, 4, 8]))
        nh = nkv * int(rng.choice([1, 3, 7, 40]))
        n, T = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 14))
        new, L = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 17))
        cap = most(nkv, nh, n, T, new, L)
        assert cap > 0
        cfg = aoship._KVConfig(1, nkv, 64, 64, 1, 0)
        for _ in range(5):
            s = [int(rng.integers(1, v + 1)) for v in (n, T, new, L)]
            b = aoship._KVBatch(s[0], s[1], s[2], s[3], P, P, P, 1 << 20)
            w = aoship._KVWeights(None, 0, 0, P, nkv * s[3], s[3])
            size = C.c_size_t()
            assert need(C.byref(cfg), 0, C.byref(b), P, 64 * nh, nh, 1.0, 0, C.byref(w), C.byref(size)) == 0
            assert 0 < size.value <= cap, (nkv, nh, n, T, new, L, s)


def _evict(layer=0, batch=None, null=False, **kw):
    d = dict(weights=P, weights_seq=2560, weights_head=640, keep=P, max_keep=300, first=4, recent=10, to_pages=P, to_stride=5,
             kept=P, kept_seq=1200, kept_head=300, weights_out=2 * P, out_seq=2560, out_head=640)
    d.update(kw)
    f = _fn("aoship_internal_kv_evict_check", [V, I, V, V])
    e = aoship._KVEvict(**d)
    return f(C.byref(CFG), layer, C.byref(batch or _batch()), None if null else C.byref(e))


def test_evict_accepts():
    assert _evict() == 0 and _evict(weights_out=None) == 0 and _evict(first=0, recent=0) == 0
    assert _evict(batch=_batch(starts=None, n_tokens=-1, max_new=-1)) == 0  # (not used)
    assert _evict(max_keep=0, to_pages=None, kept=None, to_stride=0) == 0
    assert _evict(max_keep=5000, to_stride=10, kept_seq=2560, kept_head=640) == 0  # (no more than max_len)
    assert _evict(batch=_batch(n_seqs=0)) == 1 and _evict(batch=_batch(max_len=0)) == 1


@pytest.mark.parametrize("kw", [dict(null=True), dict(layer=2), dict(layer=-1), dict(batch=_batch(n_seqs=-1)),
                                dict(batch=_batch(max_len=-1)), dict(batch=_batch(max_len=641)), dict(batch=_batch(lens=None)),
                                dict(batch=_batch(pages=None)), dict(batch=_batch(lens=P + 2)), dict(batch=_batch(page_stride=9)),
                                dict(batch=_batch(n_seqs=(1 << 20) + 1)), dict(max_keep=-1), dict(max_keep=(1 << 30) + 1),
                                dict(first=-1), dict(recent=-1), dict(keep=None), dict(keep=P + 1), dict(to_pages=None),
                                dict(to_pages=P + 2), dict(to_stride=4), dict(to_stride=-1), dict(kept=None), dict(kept=P + 2),
                                dict(kept_head=299), dict(kept_seq=1199), dict(weights=None), dict(weights=P + 1),
                                dict(weights_head=639), dict(weights_seq=2559), dict(weights_out=P), dict(weights_out=P + 6),
                                dict(out_head=639), dict(out_seq=2559)],
                         ids=lambda k: "-".join(k))
def test_evict_refuses(kw):
    assert _evict(**kw) == -1
    assert aoship.last_error().startswith("aoship_kv_evict")


def test_null_caches():
    L = aoship.lib()
    for call in (lambda: L.aoship_kv_append_at(None, 0, None, None, None, 0), lambda: L.aoship_kv_weigh_reserve(None, 1, 1, 1, 1, 1),
                 lambda: L.aoship_kv_weigh(None, 0, None, None, 0, 1, 1.0, 0, None), lambda: L.aoship_kv_evict(None, 0, None, None),
                 lambda: L.aoship_kv_cache_set_rope_axes(None, None, 0)):
        assert call() == -1 and "null cache" in aoship.last_error()
