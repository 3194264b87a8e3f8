"""CPU checks of the paged key/value cache: what its calls refuse, with every bound on both sides, how a batch's rows
are dealt to blocks of 16 positions, and the tests' own plain forms."""
import ctypes as C

import numpy as np
import pytest

import aoship
import kv_plain as P

I, V = C.c_int, C.c_void_p
ALIGNED = 1 << 12  # any aligned address: nothing is read


def _fn(name, args):
    f = getattr(aoship.lib(), name)
    f.restype, f.argtypes = I, args
    return f


CFG = aoship._KVConfig(2, 4, 128, 64, 100, 0)


def _batch(**kw):
    d = dict(n_seqs=3, n_tokens=40, max_new=20, max_len=640, starts=ALIGNED, lens=ALIGNED, pages=ALIGNED, page_stride=10)
    d.update(kw)
    return aoship._KVBatch(**d)


def _rows(**kw):
    d = dict(q=ALIGNED, k=ALIGNED, v=ALIGNED, q_stride=1024, k_stride=512, v_stride=512, q_out=2 * ALIGNED,
             q_out_stride=1024, num_heads=8)
    d.update(kw)
    return aoship._KVRows(**d)


def _append(cfg=CFG, layer=0, batch=None, rows=None, rope=0):
    f = _fn("aoship_internal_kv_append_check", [V, I, I, V, V])
    b, r = batch or _batch(), rows or _rows()
    return f(C.byref(cfg), rope, layer, C.byref(b), C.byref(r))


def _read(batch=None, k=ALIGNED, ks=512, v=ALIGNED, vs=512, layer=0):
    f = _fn("aoship_internal_kv_read_check", [V, I, V, V, C.c_int64, V, C.c_int64])
    return f(C.byref(CFG), layer, C.byref(batch or _batch()), k, ks, v, vs)


def _attention(batch=None, q=ALIGNED, qs=1024, nh=8, scale=0.1, window=0, out=2 * ALIGNED, os=1024, layer=1):
    f = _fn("aoship_internal_kv_attention_check", [V, I, V, V, C.c_int64, I, C.c_float, I, V, C.c_int64])
    return f(C.byref(CFG), layer, C.byref(batch or _batch()), q, qs, nh, scale, window, out, os)


def test_good_calls_pass():
    assert _append() == 0 and _read() == 0 and _attention() == 0
    assert _append(rows=_rows(q=None, q_out=None, num_heads=0)) == 0
    assert _append(rows=_rows(q_out=ALIGNED)) == 0  # queries rotated in place
    assert _append(rope=640) == 0


BAD_BATCHES = [dict(n_seqs=-1), dict(n_tokens=-1), dict(max_new=-1), dict(max_len=-1), dict(max_len=641),
               dict(starts=None), dict(lens=None), dict(pages=None), dict(starts=ALIGNED + 2), dict(pages=ALIGNED + 1),
               dict(page_stride=9), dict(page_stride=-1), dict(max_len=(1 << 30) + 1, page_stride=1 << 25),
               dict(n_seqs=(1 << 20) + 1), dict(n_tokens=(1 << 26) + 1)]


@pytest.mark.parametrize("kw", BAD_BATCHES, ids=lambda k: "-".join(k))
def test_bad_batches_are_refused(kw):
    for call in (_append, _read, _attention):
        assert call(batch=_batch(**kw)) == -1
        assert aoship.last_error().startswith("aoship_kv_")


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(n_tokens=0), dict(max_new=0)], ids=lambda k: "-".join(k))
def test_empty_batches_have_nothing_to_do(kw):
    for call in (_append, _read, _attention):
        assert call(batch=_batch(**kw)) == 1
    assert _attention(batch=_batch(**kw), window=-1) == -1  # (bad arguments are refused all the same)


def test_a_batch_without_positions_needs_no_pages():
    assert _attention(batch=_batch(max_len=0, pages=None, page_stride=0)) == 0


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(k=ALIGNED + 8), dict(k_stride=504), dict(v_stride=516),
                                dict(q_stride=1016), dict(q_out=None), dict(q=None), dict(num_heads=6),
                                dict(num_heads=-4), dict(num_heads=65540), dict(q_out=ALIGNED, q_out_stride=1032),
                                dict(q_out=ALIGNED + 2), dict(q_bias=ALIGNED + 4), dict(k_stride=1 << 40),
                                dict(v_bias=ALIGNED + 8)], ids=lambda k: "-".join(k))
def test_bad_rows_are_refused(kw):
    assert _append(rows=_rows(**kw)) == -1
    assert aoship.last_error().startswith("aoship_kv_append")


def test_other_refusals():
    assert _append(layer=2) == -1 and _append(layer=-1) == -1 and _read(layer=2) == -1 and _attention(layer=2) == -1
    assert _append(rope=639) == -1 and "rotary" in aoship.last_error()
    assert _read(k=None) == -1 and _read(vs=500) == -1 and _read(v=ALIGNED + 4) == -1
    assert _attention(nh=6) == -1 and _attention(nh=0) == -1 and _attention(window=-1) == -1
    assert _attention(scale=float("nan")) == -1 and _attention(scale=float("inf")) == -1
    assert _attention(out=ALIGNED) == -1 and _attention(out=None) == -1 and _attention(os=1020) == -1


def test_batches_whose_work_cannot_be_counted():
    big = dict(max_len=1 << 30, page_stride=1 << 24)
    assert _attention(batch=_batch(n_seqs=1, n_tokens=1, max_new=1, **big)) == 0
    assert _attention(batch=_batch(n_seqs=64, n_tokens=64, max_new=1, **big)) == -1 and "too large" in aoship.last_error()
    assert _append(batch=_batch(n_seqs=64, n_tokens=64, max_new=1, **big)) == 0  # (attention only)
    assert _attention(batch=_batch(n_seqs=1, n_tokens=1 << 20, max_new=1 << 20, max_len=1 << 20, page_stride=1 << 14)) == 0
    assert _attention(batch=_batch(n_seqs=1, n_tokens=1 << 26, max_new=1 << 26, max_len=1 << 26, page_stride=1 << 20)) == -1


def test_shapes_that_a_cache_refuses():
    for bad in (dict(num_layers=0), dict(num_kv_heads=0), dict(num_kv_heads=4097), dict(head_dim=0), dict(head_dim=12),
                dict(head_dim=264), dict(page_size=32), dict(page_size=96), dict(page_size=512), dict(num_pages=0),
                dict(format=3), dict(format=-1), dict(num_pages=2 ** 31 - 1, num_layers=1000)):
        c = aoship._KVConfig(2, 4, 128, 64, 100, 0)
        for n, v in bad.items():
            setattr(c, n, v)
        assert not aoship.lib().aoship_kv_cache_new(C.byref(c)), bad
        assert aoship.last_error().startswith("aoship_kv_cache_new"), bad
    assert not aoship.lib().aoship_kv_cache_new(None)
    L = aoship.lib()
    for call in (lambda: L.aoship_kv_append(None, 0, None, None), lambda: L.aoship_kv_read(None, 0, None, None, 0, None, 0),
                 lambda: L.aoship_kv_attention(None, 0, None, None, 0, 1, 1.0, 0, None, 0),
                 lambda: L.aoship_kv_cache_set_rope(None, None, None, 0), lambda: L.aoship_kv_cache_set_stream(None, None),
                 lambda: L.aoship_kv_cache_faults(None)):
        assert call() == -1 and "null cache" in aoship.last_error()
    L.aoship_kv_cache_free(None)
    with pytest.raises(aoship.AosError):
        aoship.KVCache(1, 1, 64, 64, 1, "int8")


@pytest.mark.parametrize("seed", range(40))
def test_blocks_cover_every_row_once(seed):
    """Random batches (single rows, empty sequences, padding in front, rows past the last sequence): the blocks of the
    grid, found as the launch finds them, hold every row that has a position exactly once, aligned and in their page."""
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 150))
    top = int(rng.choice([1, 2, 17, 70]))
    new = rng.integers(0, top + 1, n)
    past = rng.integers(0, 300, n) * rng.integers(0, 2, n)
    lens = np.maximum(0, past + new - (rng.random(n) < 0.1) * rng.integers(0, 40, n))
    starts = np.concatenate([[0], np.cumsum(new)])
    T, most = int(starts[-1] + rng.integers(0, 30)), max(1, int(new.max()))
    blocks = _fn("aoship_internal_kv_blocks", [I, I, I])(most, n, T)
    f = _fn("aoship_internal_kv_block", [I, I, I, I, I, I, V, V])
    base, out = C.c_int(), (C.c_int * 4)()
    found = np.zeros(T, int)
    bases = []
    for s in range(n):
        f(most, s, int(starts[s]), int(new[s]), int(lens[s]), 0, C.byref(base), out)
        bases.append(base.value)
    for x in range(blocks):
        s = int(np.searchsorted(bases, x, side="right")) - 1
        if s < 0 or not f(most, s, int(starts[s]), int(new[s]), int(lens[s]), x, C.byref(base), out):
            continue
        pos, lo, hi, row = out
        first = int(lens[s] - new[s])
        assert pos % 16 == 0 and 0 <= lo < hi <= 16 and pos + hi <= lens[s]
        assert row - starts[s] == pos + lo - first and 0 <= row - starts[s] and row + hi - lo <= starts[s + 1]
        found[row:row + hi - lo] += 1
    want = np.zeros(T, int)
    for s in range(n):
        skip = max(0, int(new[s] - lens[s]))
        want[starts[s] + min(skip, new[s]):starts[s + 1]] = 1
    assert (found == want).all()


def test_plain_quantiser():
    """The plain form against a search over every code and scale."""
    rng = np.random.default_rng(3)
    for fmt, top, codes in (("mxfp4", 6.0, [0, .5, 1, 1.5, 2, 3, 4, 6]),
                            ("mxfp8", 448.0, [m / 8 * 2.0 ** -6 for m in range(8)] +
                             [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1])):
        codes = np.array(codes)
        x = P.bf16(rng.standard_normal((50, 40)) * 2.0 ** rng.integers(-20, 20, (50, 1)))
        x[0] = 0
        x[1, 3], x[2, 35] = np.inf, np.nan
        x[3, :3] = P.bf16(np.array([top, top / 2, 2 * top]))
        got = P.quantised(x, fmt)
        for r in range(50):
            for b in (0, 32):
                blk = x[r, b:b + 32]
                if not np.isfinite(blk).all():
                    assert np.isnan(got[r, b:b + 32]).all()
                    continue
                e = next(e for e in range(-126, 130) if np.abs(blk).max() <= top * 2.0 ** e)
                e = max(e, -117 if fmt == "mxfp8" else -125)
                for i, v in enumerate(blk):
                    d = np.abs(codes * 2.0 ** e - abs(v))
                    near = np.flatnonzero(d == d.min())
                    best = near[0] if len(near) == 1 else near[near % 2 == 0][0]  # ties to the even code
                    assert abs(got[r, b + i]) == codes[best] * 2.0 ** e
                    assert got[r, b + i] == 0 or np.sign(got[r, b + i]) == np.sign(v)


# ---- the row tiles that the second attention kernel's workgroups share ----


def _pieces(nh, nkv, starts, lens, n_tokens, max_new, max_len, window=0, few=0, G=512, min_share=6, cap=1 << 16):
    """The kernel's walk over a batch, as rows of (workgroup, head, sequence, first row, rows, first position tile,
    position tiles, j, je, wf, wl), or None where it refuses the batch."""
    starts, lens = np.asarray(starts, np.int32), np.asarray(lens, np.int32)
    out = np.zeros((cap, 11), np.int32)
    f = _fn("aoship_internal_kv_tile_pieces", [I, I, I, I, I, I, I, V, V, I, I, I, V, I])
    n = f(nh, nkv, window, len(lens), n_tokens, max_new, max_len, starts.ctypes.data, lens.ctypes.data, few, G,
          min_share, out.ctypes.data, cap)
    assert n <= cap
    return None if n < 0 else out[:n]


def _row_tiles(nh, nkv, starts, lens, window, few):
    """(head, sequence, first row, rows, first position tile, position tiles) of the sequences that fit (None: those that do not), by definition"""
    g, found = nh // nkv, []
    for s, n in enumerate(lens):
        count = starts[s + 1] - starts[s]
        if n is None or count * g <= few:
            continue
        for r0 in range(0, count * g, 128):
            rows = min(128, count * g - r0)
            first, last = n - count + r0 // g, n - count + (r0 + rows - 1) // g
            t0 = max(0, first - window + 1) // 64 if window else 0
            found += [(h, s, r0, rows, t0, max(0, last) // 64 - t0 + 1) for h in range(nkv)]
    return sorted(found)


def _check_pieces(got, want):
    """Every row tile's position tiles are taken once, and each piece of a cut one expects the arrivals that come."""
    tiles = {}
    for w, h, s, r0, rows, t0, nt, j, je, wf, wl in got.tolist():
        tiles.setdefault((h, s, r0, rows, t0, nt), []).append((j, je, w, wf, wl))
    assert sorted(tiles) == want
    borders = set()
    for (_, _, _, _, _, nt), parts in tiles.items():
        parts.sort()
        assert [a for a, *_ in parts] == [0] + [b for _, b, *_ in parts[:-1]] and parts[-1][1] == nt
        if len(parts) == 1:
            assert parts[0][3:] == (-1, -1)
            continue
        wf, wl = parts[0][3:]
        assert all(p[3:] == (wf, wl) for p in parts) and len(parts) == wl - wf + 2
        assert [p[2] for p in parts] == list(range(wf - 1, wl + 1))  # their slots of the workspace
        assert not borders & set(range(wf, wl + 1))
        borders |= set(range(wf, wl + 1))


@pytest.mark.parametrize("seed", range(40))
def test_workgroups_share_row_tiles(seed):
    """Random batches: no rows, few, many, padding in front, windows, rows behind the last sequence, a sequence that
    does not fit."""
    rng = np.random.default_rng(seed)
    n, nkv, g = int(rng.integers(1, 40)), int(rng.integers(1, 5)), int(rng.choice([1, 3, 7, 16]))
    new = rng.integers(0, int(rng.choice([3, 40, 700])) + 1, n)
    lens = np.maximum(0, new + rng.integers(0, 5000, n) * rng.integers(0, 2, n) - (rng.random(n) < 0.1) * 30)
    starts, few = np.concatenate([[0], np.cumsum(new)]), int(rng.choice([0, 16]))
    window, most = int(rng.choice([0, 1, 300, 2048])), max(1, int(new.max()))
    T, max_len, fits = int(starts[-1] + rng.integers(0, 30)), int(lens.max()) + 1, list(lens)
    if rng.random() < 0.3:
        bad = int(rng.integers(0, n))
        lens[bad], fits[bad] = max_len + 5, None
    got = _pieces(g * nkv, nkv, starts, lens, T, most, max_len, window, few, G=int(rng.choice([256, 512])))
    _check_pieces(got, _row_tiles(g * nkv, nkv, starts, fits, window, few))


def test_row_tiles_of_more_rows_than_32_bits_count():
    """A batch made for 60 000 000 rows of 40 heads that holds one sequence of 1000: its row tiles and no others."""
    b = _batch(n_seqs=1, n_tokens=60000000, max_new=1000, max_len=1000, page_stride=16)
    cfg = aoship._KVConfig(1, 1, 128, 64, 100, 0)
    f = _fn("aoship_internal_kv_attention_check", [V, I, V, V, C.c_int64, I, C.c_float, I, V, C.c_int64])
    assert f(C.byref(cfg), 0, C.byref(b), ALIGNED, 5120, 40, 0.1, 0, 2 * ALIGNED, 5120) == 0
    got = _pieces(40, 1, [0, 1000], [1000], 60000000, 1000, 1000)
    _check_pieces(got, _row_tiles(40, 1, [0, 1000], [1000], 0, 0))


FALLING = [([1330, 210, 160, 610, 870], [3200, 3500, 3000, 800], 1500), ([0, 700, 300, 1000], [900, 900, 900], 1000),
           ([500, 0, 400], [600, 600], 500)]


@pytest.mark.parametrize("starts,lens,T", FALLING)
def test_starts_that_fall_are_refused_whole(starts, lens, T):
    """Which sequence a slot of row tiles belongs to would depend on where a walk comes from: workgroups that share a
    row tile would expect other arrivals than come."""
    assert _pieces(28, 4, starts, lens, T, T, 4000) is None


@pytest.mark.parametrize("starts,good", [([-2 ** 31, -2 ** 30, -9, 0, 400, 900, 950], [3, 4, 5]),
                                         ([0, 400, 900, 2 ** 30, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], [0, 1]),
                                         ([-5, 300, 300, 340, 2000, 2000, 2000], [1, 2]),
                                         ([-2 ** 31, -10 ** 8, 0, 400, 900, 950, 950], [2, 3, 4, 5])])
@pytest.mark.parametrize("g", [7, 4096])
def test_starts_outside_the_rows_leave_the_others(starts, good, g):
    """Ascending starts of which some are no rows of the batch: those sequences are left out, the others served."""
    lens = [500, 610, 600, 700, 900, 64]
    got = _pieces(2 * g, 2, starts, lens, 1000, 1000, 1000)
    _check_pieces(got, _row_tiles(2 * g, 2, starts, [n if s in good else None for s, n in enumerate(lens)], 0, 0))


def test_rotated_rows_need_no_tables():
    assert C.sizeof(aoship._KVRows) == 96
    assert _append(rope=639) == -1 and _append(rope=639, rows=_rows(rotated=1)) == 0


class _Tensor:
    """What KVBatch looks at of an int32 tensor on a device."""

    def __init__(self, device, *shape):
        import torch

        self.dtype, self.is_cuda, self.shape, self.device = torch.int32, True, shape, device

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def stride(self, i):
        return 1 if i in (-1, len(self.shape) - 1) else self.shape[-1]

    def data_ptr(self):
        return ALIGNED

    def get_device(self):
        return self.device


def test_a_batch_is_on_one_device():
    aoship.KVBatch(_Tensor(1, 4), _Tensor(1, 3), _Tensor(1, 3, 8), 5, 500)
    for devices in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(aoship.AosError, match="device"):
            aoship.KVBatch(*(_Tensor(d, *s) for d, s in zip(devices, ((4,), (3,), (3, 8)))), 5, 500)


def test_bounds_beyond_the_rows():
    """max_new bounds a sequence's rows: any number past n_tokens bounds them as n_tokens does."""
    assert _attention(batch=_batch(max_new=2 ** 31 - 1)) == 0
    assert _read(batch=_batch(max_new=2 ** 31 - 1)) == 0 and _append(batch=_batch(max_new=2 ** 31 - 1)) == 0


def test_scales_that_overflow():
    """Scores are taken in powers of two: a scale whose product with log2 e is no float32 would make every score NaN."""
    for s in (2.4e38, -2.4e38, 3.4e38):
        assert _attention(scale=s) == -1 and "scale" in aoship.last_error()
    assert _attention(scale=2.3e38) == 0 and _attention(scale=-2.3e38) == 0
