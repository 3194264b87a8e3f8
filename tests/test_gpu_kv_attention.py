"""Attention over the paged cache against float64 (tests/kv_plain.py: attention and the bound attention_bound derives
for a result: the roundings of the output and of the probabilities to bfloat16, float32 scores and sums)."""
import numpy as np
import pytest

import kv_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=[True, False], ids=["small", "large"])
def kernels(request, hip, monkeypatch):
    """Every test with the kernels that its sizes choose, and with those of large batches."""
    if not request.param:
        class Large(hip.KVCache):
            def __init__(self, *a):
                super().__init__(*a)
                self.set_small_batches(False)

        monkeypatch.setattr(hip, "KVCache", Large)


def _setup(hip, fmt, nh, nkv, hd, page, new, lens, seed=0, sharp=1.0, poison=None):
    """A cache of sequences whose rows are random, and queries for their last `new` positions."""
    rng = np.random.default_rng(seed)
    held = [max(0, n) for n in lens]
    pool = P.Pool(hip, held, nkv, hd, page, fmt, seed=seed)
    k, v = (P.bf16(rng.standard_normal((sum(held), nkv, hd))) for _ in range(2))
    if poison:
        poison(k, v)
    if sum(held):
        pool.cache.append(0, pool.batch(held, held), P.to_gpu(k), P.to_gpu(v))
    q = P.bf16(sharp * rng.standard_normal((sum(new), nh, hd)))
    cut = np.cumsum(held)[:-1]
    seqs = list(zip(np.split(q, np.cumsum(new)[:-1]), np.split(P.quantised(k, fmt), cut), np.split(P.quantised(v, fmt), cut)))
    return pool, q, seqs


def _run(pool, q, new, lens, window=0, scale=None, **kw):
    import torch

    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    pool.cache.attention(0, pool.batch(new, lens, **kw), P.to_gpu(q), out, scale=scale, window=window)
    return P.to_cpu(out)


def _check(got, seqs, new, scale, window=0):
    at = 0
    for (q, k, v), n in zip(seqs, new):
        o, a = P.attention(q, k, v, scale, window)
        g = got[at:at + n]
        at += n
        if not n:
            continue
        assert np.array_equal(np.isnan(g), np.isnan(o)), "NaN"
        tol = P.attention_bound(q, k, a, o, scale)
        fin = np.isfinite(o)
        assert np.array_equal(g[~fin & ~np.isnan(o)], o[~fin & ~np.isnan(o)])
        off = np.abs(g - o)[fin] / tol[fin]
        assert off.size == 0 or off.max() <= 1.0, (float(off.max()), n, k.shape)


ONES = [1, 2, 63, 64, 65, 128, 200, 1000]


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", [(14, 2, 64, 64), (28, 4, 128, 128), (3, 3, 128, 64), (40, 1, 80, 64),
                                            (4, 2, 256, 256), (6, 2, 8, 64), (5, 1, 136, 64)])
def test_one_token_each(hip, fmt, nh, nkv, hd, page):
    """Lengths about the tiles' borders, more query heads than a matrix instruction has columns, none."""
    new = [1] * len(ONES) + [0]
    lens = ONES + [77]
    pool, q, seqs = _setup(hip, fmt, nh, nkv, hd, page, new, lens, seed=hd)
    _check(_run(pool, q, new, lens), seqs, new, hd ** -0.5)
    assert pool.cache.faults() == 0


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", [(14, 2, 64, 64), (7, 1, 128, 64), (2, 2, 128, 128), (3, 1, 80, 64), (8, 2, 256, 64)])
@pytest.mark.parametrize("window", [0, 1, 70])
def test_chunks(hip, fmt, nh, nkv, hd, page, window):
    """Drafted tokens, chunks over what is held, whole prompts and single tokens in one call."""
    new = [3, 65, 1, 130, 16, 0, 40]
    past = [100, 0, 300, 64, 0, 5, 171]
    lens = [a + b for a, b in zip(new, past)]
    pool, q, seqs = _setup(hip, fmt, nh, nkv, hd, page, new, lens, seed=hd + window)
    _check(_run(pool, q, new, lens, window), seqs, new, hd ** -0.5, window)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", [(14, 2, 64, 64), (28, 4, 128, 128), (6, 1, 80, 64), (12, 2, 256, 64)])
@pytest.mark.parametrize("window", [0, 33])
def test_drafted(hip, fmt, nh, nkv, hd, page, window):
    """Up to 28 rows a sequence: one and two blocks of a matrix instruction's columns, the second in part or empty."""
    new = [4, 1, 3, 0, 2, 4]
    lens = [70, 1, 3, 9, 700, 64]
    pool, q, seqs = _setup(hip, fmt, nh, nkv, hd, page, new, lens, seed=hd + window)
    _check(_run(pool, q, new, lens, window), seqs, new, hd ** -0.5, window)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("new,lens", [([1], [9001]), ([3], [30001]), ([5], [20011]), ([300], [3001]), ([700], [700]),
                                      ([1, 1], [64, 40000])])
def test_long(hip, fmt, new, lens):
    """Row tiles that many workgroups share, and uneven lengths."""
    pool, q, seqs = _setup(hip, fmt, 7, 1, 128, 256, new, lens, seed=lens[-1], sharp=3.0)
    got = _run(pool, q, new, lens)
    _check(got, seqs, new, 128 ** -0.5)
    for _ in range(3):
        assert np.array_equal(got, _run(pool, q, new, lens))  # (no order depends on timing)


@pytest.mark.parametrize("n,new", [(150, 1), (70, 2), (130, 20)])
def test_many_sequences(hip, n, new):
    """More sequences than lanes, some without rows or positions."""
    rng = np.random.default_rng(n)
    news = [int(x) for x in rng.integers(0, new + 1, n)]
    lens = [a + int(b) for a, b in zip(news, rng.integers(0, 200, n))]
    pool, q, seqs = _setup(hip, "mxfp8", 4, 2, 64, 64, news, lens)
    _check(_run(pool, q, news, lens, max_new=new), seqs, news, 64 ** -0.5)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("new,lens", [([6, 4, 1], [2, 0, 0]), ([12, 16, 2], [9, 3, 0]), ([40, 90, 3], [10, 70, 0])])
def test_rows_that_see_nothing(hip, fmt, new, lens):
    """Sequences padded in front, and rows of a sequence without positions: zeros."""
    pool, q, seqs = _setup(hip, fmt, 4, 2, 128, 64, new, lens)
    got = _run(pool, q, new, lens)
    _check(got, seqs, new, 128 ** -0.5)
    assert (got[:new[0] - lens[0]] == 0).all() and (got[-new[2]:] == 0).all()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 80, 79])
def test_windows_past_everything(hip, window):
    """Windows as long as the sequence or longer, with rows in front that have no position."""
    new, lens = [12, 90, 1], [7, 80, 80]
    pool, q, seqs = _setup(hip, "bf16", 4, 2, 64, 64, new, lens)
    _check(_run(pool, q, new, lens, window), seqs, new, 64 ** -0.5, window)


@pytest.mark.parametrize("fmt,new", [("bf16", 1), ("bf16", 20), ("mxfp8", 1), ("mxfp8", 20)])
def test_far_pages(hip, fmt, new):
    """Pages whose offset passes 32 bits, in the last layer of a cache of more than 4 GB a layer."""
    import torch

    rng = np.random.default_rng(1)
    nh, nkv, hd, L, page = 8, 8, 128, 300, 256
    row = 2 * nkv * (hd * 2 if fmt == "bf16" else hd + hd // 32)
    n = (1 << 32) // (row * page) + 8
    cache = hip.KVCache(2, nkv, hd, page, n, fmt)
    pages = torch.tensor([[n - 1, n - 3]], dtype=torch.int32).cuda()
    k, v = (P.bf16(rng.standard_normal((L, nkv, hd))) for _ in range(2))
    q = P.bf16(rng.standard_normal((new, nh, hd)))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    cache.append(1, hip.KVBatch(i32(0, L), i32(L), pages, L, L), P.to_gpu(k), P.to_gpu(v))
    out = torch.empty((new, nh, hd), dtype=torch.bfloat16, device="cuda")
    cache.attention(1, hip.KVBatch(i32(0, new), i32(L), pages, new, L), P.to_gpu(q), out)
    _check(P.to_cpu(out), [(q, P.quantised(k, fmt), P.quantised(v, fmt))], [new], hd ** -0.5)
    back = [torch.empty((L, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.read(1, hip.KVBatch(i32(0, L), i32(L), pages, L, L), *back)
    assert np.array_equal(P.to_cpu(back[0]), P.quantised(k, fmt)) and np.array_equal(P.to_cpu(back[1]), P.quantised(v, fmt))
    assert cache.faults() == 0


@pytest.mark.parametrize("new", [1, 3, 30])
def test_two_caches_at_once(hip, new):
    """Two caches' calls on two streams at the same time: each has its own workspace."""
    import torch

    lens = [3000 + new, 5000 + new]
    made = [_setup(hip, f, 8, 1, 128, 64, [new] * 2, lens, seed=i) for i, f in enumerate(("mxfp8", "bf16"))]
    streams = [torch.cuda.Stream() for _ in made]
    outs, runs = [], []
    for (pool, q, _), st in zip(made, streams):
        outs.append(torch.empty(q.shape, dtype=torch.bfloat16, device="cuda"))
        runs.append((pool, pool.batch([new] * 2, lens), P.to_gpu(q), outs[-1]))
        pool.cache.set_stream(st.cuda_stream)
    torch.cuda.synchronize()
    for _ in range(10):
        for pool, batch, q, out in runs:
            pool.cache.attention(0, batch, q, out)
    torch.cuda.synchronize()
    for (_, _, seqs), out in zip(made, outs):
        _check(P.to_cpu(out), seqs, [new] * 2, 128 ** -0.5)


def test_pages_shared_by_readers(hip):
    """Sequences with a common prefix read the same pages."""
    import torch

    new, L, nh, hd = [1, 1, 60], 190, 4, 64
    pool, q, seqs = _setup(hip, "mxfp8", nh, 2, hd, 64, [1], [L])
    pool.pages = pool.pages.expand(3, -1).contiguous()
    rng = np.random.default_rng(8)
    q = P.bf16(rng.standard_normal((62, nh, hd)))
    _, k, v = seqs[0]
    lens = [130, L, 128]
    _check(_run(pool, q, new, lens), [(q[:1], k[:130], v[:130]), (q[1:2], k, v), (q[2:], k[:128], v[:128])], new, hd ** -0.5)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("new", [1, 4, 14, 90])
def test_infinities_and_nans(hip, fmt, new):
    """Visible ones reach the rows that see them, by the formula; those of later positions, of positions left of the
    window and of stale rows in a page reach nobody."""
    nh, nkv, hd, L = 4, 2, 64, 230
    first = L - new

    def poison(k, v):
        v[first + new // 2, 0, 5] = np.inf       # seen by the second half of the new rows
        v[first + new // 2, 0, 6] = -np.inf
        v[L - 1, 1, 40] = np.nan                 # seen by the last row only
        k[L - 1, 1, 33] = np.nan if new > 1 else 0.0
        v[2, :, :] = np.nan                      # left of every window
        k[3, :, :] = np.inf
        v[L:] = np.nan                           # (stale rows: written by an earlier, longer sequence)
        k[L:] = np.nan

    pool, q, seqs = _setup(hip, fmt, nh, nkv, hd, 64, [new], [L + 20], poison=poison)
    q, (_, k, v) = q, seqs[0]
    got = _run(pool, q, [new], [L], window=100, max_len=256)
    want = [(q, k[:L], v[:L])]
    if fmt == "bf16":
        _check(got, want, [new], hd ** -0.5, 100)
    else:  # a block of 32 dimensions is NaN whole: compare where the float64 form is finite, and its NaNs
        o, a = P.attention(q, k[:L], v[:L], hd ** -0.5, 100)
        assert np.array_equal(np.isnan(got), ~np.isfinite(o))
        fin = np.isfinite(o)
        assert (np.abs(got - o)[fin] <= P.attention_bound(q, k[:L], a, o, hd ** -0.5)[fin]).all()


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("new", [2, 12, 90])
def test_largest_values(hip, fmt, new):
    """A value whose code stands for 2^128 is an infinity to the row that sees it, and nothing to the others."""
    def poison(k, v):
        v[229, 1, 40] = P.bf16([3.3895e38])[0]
        k[229] = 0.0

    pool, q, seqs = _setup(hip, fmt, 4, 2, 64, 64, [new], [230], poison=poison)
    got = _run(pool, q, [new], [230])
    o, a = P.attention(*seqs[0], 64 ** -0.5)
    assert (np.abs(got - o)[:-1] <= P.attention_bound(seqs[0][0], seqs[0][1], a, o, 64 ** -0.5)[:-1]).all()


@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (14, 2, 128), (2, 1, 256)])
def test_infinite_scores(hip, nh, nkv, hd):
    """Scores of plus infinity make their rows NaN, and so do scores of minus infinity where a row sees no others."""
    new, lens = [1, 70, 1, 1, 3, 40], [1, 70, 200, 300, 700, 700]

    def poison(k, v):
        k[0, :, 0] = np.inf             # the only position of the first sequence
        k[1, :, 0] = -np.inf            # the first position of the second
        k[71 + 150:71 + 200, :, 1] = np.inf   # the last positions of the third
        k[271:, :, 2] = np.inf          # every position of the others
        k[1271 + 600, :, 2] = 1.0       # but one

    pool, q, seqs = _setup(hip, "bf16", nh, nkv, hd, 64, new, lens, seed=hd, poison=poison)
    _check(_run(pool, q, new, lens), seqs, new, hd ** -0.5)


@pytest.mark.parametrize("sharp,scale", [(60.0, None), (1.0, 0.0), (2.0, -0.3)])
def test_scores_of_any_size(hip, sharp, scale):
    """Scores of hundreds (the running maximum moves far), a scale of zero, a negative one."""
    new, lens = [1, 30], [500, 400]
    pool, q, seqs = _setup(hip, "bf16", 4, 2, 64, 64, new, lens, sharp=sharp)
    _check(_run(pool, q, new, lens, scale=scale), seqs, new, 64 ** -0.5 if scale is None else scale)


def test_strides_and_rows_left_alone(hip):
    """Queries as a slice of a joint projection, outputs into a wider tensor, rows behind the last sequence."""
    import torch

    new, lens, nh, hd = [1, 70, 2], [80, 90, 300], 4, 128
    pool, q, seqs = _setup(hip, "mxfp8", nh, 2, hd, 64, new, lens)
    T = sum(new)
    joint = torch.zeros((T + 5, nh + 3, hd), dtype=torch.bfloat16, device="cuda")
    joint[:T, 1:1 + nh] = P.to_gpu(q)
    wide = torch.full((T + 5, nh + 2, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    pool.cache.attention(0, pool.batch(new, lens), joint[:, 1:1 + nh], wide[:, 2:])
    _check(P.to_cpu(wide[:T, 2:]), seqs, new, hd ** -0.5)
    assert (wide[:T, :2] == 7).all() and (wide[T:] == 7).all()


def test_bad_pages_and_rows(hip):
    """Positions of a page outside the cache are not attended to; a sequence that does not fit is left alone; both are
    reported and neighbours are served."""
    import torch

    for new in ([1, 1, 1], [1, 12, 9], [1, 100, 40]):
        lens, nh, hd = [70, 200, 90], 4, 64
        pool, q, seqs = _setup(hip, "bf16", nh, 2, hd, 64, new, lens)
        pool.pages[1, 1] = 10 ** 7
        got = _run(pool, q, new, lens)
        assert pool.cache.faults() == hip.KV_FAULT_PAGE
        _check(got[:1], seqs[:1], new[:1], hd ** -0.5)
        _check(got[-new[2]:], seqs[2:], new[2:], hd ** -0.5)
        qq, k, v = seqs[1]
        for t in (0, new[1] - 1):
            end = lens[1] - new[1] + t + 1
            keep = [i for i in range(end) if not 64 <= i < 128]
            o, a = P.attention(qq[t:t + 1], k[keep], v[keep], hd ** -0.5)
            assert (np.abs(got[new[0] + t] - o[0]) <= P.attention_bound(qq, k, a, o, hd ** -0.5)[0]).all()
        pool.pages.copy_(torch.from_numpy(pool.table))
        for bad in ([70, 201, 90], [70, -3, 90]):
            got = _run(pool, q, new, bad, max_len=200)
            assert pool.cache.faults() == hip.KV_FAULT_BATCH
            assert (got[new[0]:new[0] + new[1]] == 7).all()
            _check(got[:1], seqs[:1], new[:1], hd ** -0.5)
        pool.pages[0, 0] = -1  # nothing left to see
        got = _run(pool, q, new, [64, 200, 90])
        assert (got[0] == 0).all() and pool.cache.faults() == hip.KV_FAULT_PAGE


@pytest.mark.parametrize("new", [1, 40])
def test_graph_replays(hip, new):
    """append and attention captured on another stream, replayed while the sequences grow, between eager work."""
    import torch

    rng = np.random.default_rng(new)
    n, nh, nkv, hd, cap = 4, 8, 2, 128, 900
    pool = P.Pool(hip, [cap] * n, nkv, hd, 64, "bf16")
    start = [3, 500, 64, 250]
    past = [P.bf16(rng.standard_normal((sum(start), nkv, hd))) for _ in range(2)]
    pool.cache.append(0, pool.batch(start, start), *map(P.to_gpu, past))
    held = [list(np.split(x, np.cumsum(start)[:-1])) for x in past]
    q, k, v = (torch.zeros((n * new, h, hd), dtype=torch.bfloat16, device="cuda") for h in (nh, nkv, nkv))
    out = torch.empty_like(q)
    batch = pool.batch([new] * n, [s + new for s in start], max_len=cap)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    pool.cache.set_stream(side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pool.cache.append(0, batch, k, v)
        pool.cache.attention(0, batch, q, out)
    for step in range(4):
        x = [P.bf16(rng.standard_normal(t.shape)) for t in (q, k, v)]
        for t, y in zip((q, k, v), x):
            t.copy_(P.to_gpu(y))
        if step:
            batch.lens += new
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for s in range(n):
                held[i][s] = np.concatenate([held[i][s], x[1 + i][s * new:(s + 1) * new]])
        seqs = [(x[0][s * new:(s + 1) * new], held[0][s], held[1][s]) for s in range(n)]
        _check(P.to_cpu(out), seqs, [new] * n, hd ** -0.5)
    pool.cache.set_stream(None)


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_a_layer_as_it_is_served(hip, fmt):
    """q/k/v projections with adapters, biases, rotary embedding and cache, attention, o projection: a prompt of each
    of three streams, then tokens one by one, against the same steps in float64 from the projections' outputs."""
    import torch

    rng = np.random.default_rng(9)
    hidden, nh, nkv, hd = 512, 8, 2, 64
    layer = hip.Layer(0)
    for m, o, i in (("q_proj", nh * hd, hidden), ("k_proj", nkv * hd, hidden), ("v_proj", nkv * hd, hidden),
                    ("o_proj", hidden, nh * hd)):
        layer.set_base(m, rng.integers(0, 2 ** 32, (o, i // 8), dtype=np.uint32),
                       (rng.random((o, i // 64)) * 0.01).astype(np.float16), np.full((o, i // 64), -0.04, np.float16))
    ad = hip.LoraAdapter(0, 1, 1.0)
    for m, o, i in (("q_proj", nh * hd, hidden), ("o_proj", hidden, nh * hd)):
        ad.set_module(0, m, (rng.standard_normal((16, i)) / i ** 0.5).astype(np.float32),
                      (0.01 * rng.standard_normal((o, 16))).astype(np.float32))
    layer.set_adapters([ad])
    ring = np.zeros(1, hip.RING_DTYPE)
    ring["top_k"], ring["gates_q15"][0, 0] = 1, 32767
    pool = P.Pool(hip, [150] * 3, nkv, hd, 64, fmt)
    cos, sin = (f(np.arange(150)[:, None] * 10.0 ** (-np.arange(hd // 2) / 8)).astype(np.float32) for f in (np.cos, np.sin))
    pool.cache.set_rope(cos, sin)
    bias = [rng.standard_normal((h, hd)).astype(np.float32) for h in (nh, nkv, nkv)]
    gb = [torch.from_numpy(b).cuda() for b in bias]
    kept = [[np.zeros((0, nkv, hd))] * 3 for _ in range(2)]
    lens = [0, 0, 0]
    for new in ([100, 37, 5], [1, 1, 1], [1, 1, 0], [1, 2, 9]):
        T = sum(new)
        x = P.to_gpu(rng.standard_normal((T, hidden)))
        rings = torch.from_numpy(np.repeat(ring, T).view(np.uint8)).cuda()
        q, k, v = (torch.empty((T, h, hd), dtype=torch.bfloat16, device="cuda") for h in (nh, nkv, nkv))
        layer.qkv_forward(x, rings, q, k, v)
        raw = [P.to_cpu(t) for t in (q, k, v)]
        at = list(lens)
        lens = [a + b for a, b in zip(lens, new)]
        batch = pool.batch(new, lens)
        pool.cache.append(0, batch, k, v, q=q, q_out=q, q_bias=gb[0], k_bias=gb[1], v_bias=gb[2])
        out = torch.empty_like(q)
        pool.cache.attention(0, batch, q, out)
        y = torch.empty((T, hidden), dtype=torch.bfloat16, device="cuda")
        layer.proj_forward("o_proj", out.view(T, nh * hd), rings, y)
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(at, new)])
        full = [r.astype(np.float32) + b for r, b in zip(raw, bias)]
        rows = [P.bf16(P.rotated(full[0], cos[pos], sin[pos])), P.bf16(P.rotated(full[1], cos[pos], sin[pos])), P.bf16(full[2])]
        seqs = []
        for s in range(3):
            part = slice(sum(new[:s]), sum(new[:s + 1]))
            for i in range(2):
                kept[i][s] = np.concatenate([kept[i][s], P.quantised(rows[1 + i][part], fmt)])
            seqs.append((rows[0][part], kept[0][s], kept[1][s]))
        _check(P.to_cpu(out), seqs, new, hd ** -0.5)
        again = torch.empty_like(y)
        layer.proj_forward("o_proj", out.view(T, nh * hd), rings, again)
        assert torch.isfinite(y).all() and torch.equal(y, again)
    assert pool.cache.faults() == 0


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_starts_that_fall(hip, fmt):
    """Noted, no row written, and the cache's next calls are right: workgroups that share a row tile count their
    arrivals in words that stay with the cache."""
    new, lens, nh, hd = [700, 300, 100], [900, 400, 300], 28, 64
    pool, q, seqs = _setup(hip, fmt, nh, 4, hd, 64, new, lens)
    for starts in ([0, 700, 300, 1100], [700, 0, 400, 900]):
        got = _run(pool, q, new, lens, starts=starts, max_new=1100)
        assert pool.cache.faults() == hip.KV_FAULT_BATCH and (got == 7).all()
        _check(_run(pool, q, new, lens), seqs, new, hd ** -0.5)
        assert pool.cache.faults() == 0


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
@pytest.mark.parametrize("new", [1, 3, 14, 90, 700])
def test_pages_left_of_every_window(hip, fmt, new):
    """Pages taken back (-1 in the table) since no row sees them any more are no fault; a page that one does see is."""
    L, window, nh, hd = 5000, 300, 4, 64
    pool, q, seqs = _setup(hip, fmt, nh, 2, hd, 64, [new], [L])
    gone = (L - new - window + 1) // 64
    pool.pages[0, :gone] = -1
    _check(_run(pool, q, [new], [L], window), seqs, [new], hd ** -0.5, window)
    assert pool.cache.faults() == 0
    pool.pages[0, gone] = -1
    _run(pool, q, [new], [L], window)
    assert pool.cache.faults() == hip.KV_FAULT_PAGE


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("new", [1, 7, 300])
@pytest.mark.parametrize("odd", [False, True])
def test_large_values_far_below_the_maximum(hip, fmt, new, odd):
    """A long run of positions whose scores lie hundreds below the others' counts for nothing, however large its values
    (odd: also in a cache that has held an infinity). Their scores are all the same and their probabilities beside each
    other 1: 2000 of them times 2^116 stay below 2^127."""
    L, nh, hd = 6000, 4, 128

    def poison(k, v):
        k[:2000] = 0.0
        k[:2000, :, 0] = -256.0
        v[:2000] = 2.0 ** 116
        if odd:
            v[L] = np.inf

    pool, q, seqs = _setup(hip, fmt, nh, 1, hd, 64, [new], [L + 1], poison=poison)
    q[:, :, 0] = 16.0  # (-4096 / sqrt(128) = -362 of a score)
    _, k, v = seqs[0]
    _check(_run(pool, q, [new], [L], max_len=L + 1), [(q, k[:L], v[:L])], [new], hd ** -0.5)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("hd", [80, 128, 256])
@pytest.mark.parametrize("new", [1, 4, 14, 90])
def test_infinities_and_nans_in_wide_heads(hip, fmt, hd, new):
    """As above, in dimensions of every block, and over enough positions that workgroups share a row tile: the
    marked elements are more than a word of bits there."""
    nh, nkv, L, window = 4, 2, 900, 700
    first = L - new
    dims = [d for d in (0, 5, 33, 63, 79, 95, 127, 128, 191, 255) if d < hd]

    def poison(k, v):
        for i, d in enumerate(dims):
            v[first + new // 2, 0, d] = (np.inf, -np.inf, np.nan)[i % 3]  # seen by the second half of the new rows
            v[first - 100 - 40 * i, 1, d] = (-np.inf, np.nan, np.inf)[i % 3]  # seen by all
        v[first - 333, 1, dims[-1]] = -np.inf  # (meets a plus infinity of the same dimension, or not)
        v[L - 1, 1, 1] = np.nan                # seen by the last row only
        v[:first - window + 1] = np.nan        # left of every window
        v[L:] = -np.inf                        # (stale rows)
        k[L:] = np.nan

    pool, q, seqs = _setup(hip, fmt, nh, nkv, hd, 64, [new], [L + 20], poison=poison)
    _, k, v = seqs[0]
    got = _run(pool, q, [new], [L], window=window, max_len=960)
    if fmt == "bf16":
        _check(got, [(q, k[:L], v[:L])], [new], hd ** -0.5, window)
    else:
        o, a = P.attention(q, k[:L], v[:L], hd ** -0.5, window)
        assert np.array_equal(np.isnan(got), ~np.isfinite(o))
        fin = np.isfinite(o)
        assert (np.abs(got - o)[fin] <= P.attention_bound(q, k[:L], a, o, hd ** -0.5)[fin]).all()
    assert np.array_equal(got, _run(pool, q, [new], [L], window=window, max_len=960), equal_nan=True)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("new", [2, 12, 90])
def test_largest_values_where_they_are_seen(hip, fmt, new):
    """The row that sees a value whose code stands for 2^128 takes it as that number or as infinity, the rest of its
    dimensions and the other heads as they are."""
    def poison(k, v):
        v[229, 1, 40] = P.bf16([3.3895e38])[0]
        k[229] = 0.0

    pool, q, seqs = _setup(hip, fmt, 4, 2, 64, 64, [new], [230], poison=poison)
    got = _run(pool, q, [new], [230])[-1]
    q, k, v = seqs[0]
    assert np.isinf(v).sum() == 1
    v = np.where(np.isinf(v), 2.0 ** 128, v)
    o, a = P.attention(q[-1:], k, v, 64 ** -0.5)
    near = np.abs(got - o[0]) <= P.attention_bound(q, k, a, o, 64 ** -0.5)[0]
    top = np.zeros_like(near)
    top[2:, 40] = True
    assert (near | (top & (got == np.inf))).all()


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("new,count", [(1, 96), (4, 64), (400, 5)])
@pytest.mark.parametrize("odd", [False, True])
def test_with_the_chip_full(hip, fmt, new, count, odd):
    """Waves that convert and multiply side by side on every SIMD: float64 of what the cache holds, and the same bits
    each time (odd: the bodies for caches that have held an infinity)."""
    import torch

    nh, nkv, hd = 28, 4, 128
    rng = np.random.default_rng(count)
    lens = [int(n) for n in rng.integers(1200, 2500, count)]
    pool = P.Pool(hip, [*lens, 1], nkv, hd, 64, fmt)
    gen = torch.Generator(device="cuda").manual_seed(count)
    k, v = (torch.randn((sum(lens), nkv, hd), generator=gen, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((count * new, nh, hd), generator=gen, device="cuda").bfloat16()
    pool.cache.append(0, pool.batch([*lens, 0], [*lens, 0]), k, v)
    if odd:  # (in a page of a sequence that is not among the others)
        bad = torch.full((1, nkv, hd), float("inf"), dtype=torch.bfloat16, device="cuda")
        pool.cache.append(0, pool.batch([0] * count + [1], [0] * count + [1]), bad, bad)
    pool.cache.read(0, pool.batch([*lens, 0], [*lens, 0]), k, v)
    batch = pool.batch([new] * count + [0], [*lens, 0])
    outs = [torch.empty_like(q) for _ in range(6)]
    for out in outs:
        pool.cache.attention(0, batch, q, out)
    assert pool.cache.faults() == 0
    assert all(torch.equal(out.view(torch.int16), outs[0].view(torch.int16)) for out in outs)
    at = 0
    for s, n in enumerate(lens):
        ks, vs = (x[at:at + n].double().transpose(0, 1).contiguous() for x in (k, v))
        at += n
        rows = slice(s * new, (s + 1) * new)
        qs = q[rows].double().view(new, nkv, -1, hd).permute(1, 0, 2, 3).reshape(nkv, -1, hd)
        sc = torch.matmul(qs, ks.transpose(1, 2).contiguous()) * hd ** -0.5
        hidden = torch.arange(n, device="cuda") > (n - new + torch.arange(new, device="cuda"))[:, None]
        p = torch.softmax(sc.view(nkv, new, -1, n).masked_fill(hidden[None, :, None], float("-inf")).flatten(1, 2), -1)
        o, a = torch.matmul(p, vs), torch.matmul(p, vs.abs())
        d = (hd + 4) * 2.0 ** -24 * hd ** -0.5 * qs.abs().sum(-1).max() * ks.abs().max()  # (as attention_bound)
        got = outs[0][rows].double().view(new, nkv, -1, hd).permute(1, 0, 2, 3).reshape(nkv, -1, hd)
        assert ((got - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.2 * d + 2.0 ** -14) * a + 1e-30).all()
