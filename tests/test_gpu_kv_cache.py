"""The paged cache's append and read on the GPU against the plain forms (tests/kv_plain.py). Every comparison is
exact: the rotation's float32 operations are rounded one by one in both, a power-of-two scale changes no significand,
and codes and bfloat16 values are rounded to nearest even by rule."""
import numpy as np
import pytest

import kv_plain as P

pytestmark = pytest.mark.gpu

SHAPES = [(4, 2, 64, 64), (8, 2, 128, 128), (3, 3, 80, 64), (4, 1, 8, 256), (6, 3, 256, 64), (2, 1, 136, 128)]


def _rows(rng, T, heads, hd):
    x = rng.standard_normal((T, heads, hd)) * np.exp2(rng.integers(-4, 5, (T, heads, 1)))
    return P.bf16(x)


def _same(got, want):
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


def _wanted(k, cos, sin, pos, bias, rotate):
    x = k.astype(np.float32) + (0 if bias is None else bias.astype(np.float32))
    return P.bf16(P.rotated(x, cos[pos], sin[pos]) if rotate else x)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("rope,bias", [(True, True), (False, False), (True, False)])
def test_append_and_read(hip, fmt, nh, nkv, hd, page, rope, bias):
    """Ragged sequences (no new row, one, many; at and off block and page borders) over positions held before; rows of
    a joint tensor; then everything is read back."""
    import torch

    rng = np.random.default_rng(hd + nh)
    past = [0, 5, page - 1, 16, page * 2 + 3, 0, 40]
    new = [1, 0, 20, 16, 1, 70, page + 9]
    lens = [a + b for a, b in zip(past, new)]
    pool = P.Pool(hip, lens, nkv, hd, page, fmt, layers=2)
    cache, T = pool.cache, sum(new)
    cos, sin = (f(np.arange(max(lens))[:, None] * 3.0 ** -np.arange(hd // 2)).astype(np.float32) for f in (np.cos, np.sin))
    old = [_rows(rng, sum(past), nkv, hd) for _ in range(2)]
    cache.append(1, pool.batch(past, past), *map(P.to_gpu, old))  # (no rotation yet)
    if rope:
        cache.set_rope(cos, sin)
    q, k, v = _rows(rng, T, nh, hd), _rows(rng, T, nkv, hd), _rows(rng, T, nkv, hd)
    joint = P.to_gpu(np.concatenate([q, k, v], 1))
    gq, gk, gv = joint[:, :nh], joint[:, nh:nh + nkv], joint[:, nh + nkv:]
    b = [rng.standard_normal((h, hd)).astype(np.float32) if bias else None for h in (nh, nkv, nkv)]
    gb = [None if x is None else torch.from_numpy(x).cuda() for x in b]
    wide = torch.full((T + 3, nh + 1, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    q_out = wide[:T, :nh]
    cache.append(1, pool.batch(new, lens), gk, gv, q=gq, q_out=q_out, q_bias=gb[0], k_bias=gb[1], v_bias=gb[2])
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, new)])
    _same(P.to_cpu(q_out), _wanted(q, cos, sin, pos, b[0], rope))
    assert (wide[:T, nh] == 7).all() and (wide[T:] == 7).all()

    k_now, v_now = _wanted(k, cos, sin, pos, b[1], rope), _wanted(v, cos, sin, pos, b[2], False)
    split = lambda x, n: np.split(x, np.cumsum(n)[:-1])  # noqa: E731
    whole = [P.quantised(np.concatenate([r for pair in zip(split(o, past), split(x, new)) for r in pair]), fmt)
             for o, x in zip(old, (k_now, v_now))]
    S = sum(lens)
    back = [torch.full((S + 2, nkv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.read(1, pool.batch(lens, lens), *back)
    for got, want in zip(back, whole):
        _same(P.to_cpu(got)[:S], want)
        assert (got[S:] == 7).all()  # rows behind the last sequence
    part = [torch.empty((T, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.read(1, pool.batch(new, lens), *part)
    for got, x in zip(part, (k_now, v_now)):
        _same(P.to_cpu(got), P.quantised(x, fmt))
    cache.read(0, pool.batch(lens, lens), *back)  # the other layer holds nothing
    assert all((t[:S] == 0).all() for t in back)
    assert cache.faults() == 0


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_token_by_token_equals_one_call(hip, fmt):
    import torch

    rng = np.random.default_rng(1)
    lens, nkv, hd = [37, 70], 2, 128
    k, v = (P.to_gpu(_rows(rng, sum(lens), nkv, hd)) for _ in range(2))
    a, b = (P.Pool(hip, lens, nkv, hd, 64, fmt) for _ in range(2))
    a.cache.append(0, a.batch(lens, lens), k, v)
    for i in range(max(lens)):
        new = [1 if i < n else 0 for n in lens]
        rows = torch.tensor([off + i for off, n in zip((0, 37), lens) if i < n], device="cuda")
        b.cache.append(0, b.batch(new, [min(i + 1, n) for n in lens]), k[rows].contiguous(), v[rows].contiguous())
    got = []
    for p in (a, b):
        back = [torch.empty_like(k) for _ in range(2)]
        p.cache.read(0, p.batch(lens, lens), *back)
        got.append(torch.cat(back).view(torch.int16))
    assert torch.equal(*got)


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_special_values(hip, fmt):
    """Zeros, subnormals, the largest finite values, signed zeros; infinities and NaNs keep to their own block."""
    import torch

    hd, T = 128, 24
    x = np.random.default_rng(5).standard_normal((T, 1, hd))
    x[0] = 0
    x[1] = -0.0
    x[2] *= 2.0 ** -126
    x[3] *= 2.0 ** -132
    x[4] *= 2.0 ** 126
    x[5, 0, 40], x[6, 0, 3], x[7, 0, 127] = np.inf, -np.inf, np.nan
    x[8, 0, :2] = 2.0 ** -120, 2.0 ** -133
    x[9, 0, 64:] = 0
    x = P.bf16(x)
    x[10] = np.float64(np.float32(3.3895314e38))
    pool = P.Pool(hip, [T], 1, hd, 64, fmt)
    pool.cache.append(0, pool.batch([T], [T]), P.to_gpu(x), P.to_gpu(x[::-1]))
    k, v = (torch.empty((T, 1, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pool.cache.read(0, pool.batch([T], [T]), k, v)
    _same(P.to_cpu(k), P.quantised(x, fmt))
    _same(P.to_cpu(v), P.quantised(x, fmt)[::-1])


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_padding_bad_pages_and_bad_rows(hip, fmt):
    """Rows before a sequence's first position are skipped; pages outside the cache and sequences whose rows or length
    do not fit are left out and reported; neighbours are served, and nothing else of the cache changes."""
    import torch

    rng = np.random.default_rng(2)
    nkv, hd, lens = 2, 64, [20, 100, 30, 10]
    pool = P.Pool(hip, lens, nkv, hd, 64, fmt, spare=3)
    guard = hip.KVBatch(torch.tensor([0, 64, 128, 192], dtype=torch.int32).cuda(),
                        torch.full((3,), 64, dtype=torch.int32).cuda(),
                        torch.from_numpy(pool.spare.astype(np.int32)[:, None].copy()).cuda(), 64, 64)
    fill = P.to_gpu(_rows(rng, 192, nkv, hd))
    pool.cache.append(0, guard, fill, fill)

    def whole():
        t = [torch.empty((192, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        pool.cache.read(0, guard, *t)
        return torch.cat(t)

    before = whole()
    new = [25, 100, 30, 10]  # the first sequence: five rows in front that it does not hold
    T = sum(new)
    k, v = _rows(rng, T, nkv, hd), _rows(rng, T, nkv, hd)
    pool.pages[1, 1] = 10 ** 6  # its second page
    pool.cache.append(0, pool.batch(new, lens), P.to_gpu(k), P.to_gpu(v))
    assert pool.cache.faults() == hip.KV_FAULT_PAGE
    assert pool.cache.faults() == 0
    got = [torch.full((T, nkv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pool.cache.read(0, pool.batch(new, lens), *got)
    assert pool.cache.faults() == hip.KV_FAULT_PAGE
    for g, x in zip(got, (k, v)):
        want = P.quantised(x, fmt)
        want[:5] = 7.0
        want[25 + 64:125] = 0.0
        _same(P.to_cpu(g), want)
    pool.pages[1, 1] = -5
    pool.cache.append(0, pool.batch(new, lens), P.to_gpu(k), P.to_gpu(v))
    assert pool.cache.faults() == hip.KV_FAULT_PAGE

    table = pool.table.copy()
    pool.pages.copy_(torch.from_numpy(table))
    for kw, out in ((dict(lens=[20, 100, 641, 10], max_len=128), 2), (dict(lens=[20, -1, 30, 10]), 1),
                    (dict(max_new=60), 1), (dict(starts=[0, 25, 125, 120, 130]), 2), (dict(starts=[0, 25, 125, 155, 166]), 3),
                    (dict(starts=[-1, 25, 125, 155, 165]), 0)):
        pool.cache.append(0, pool.batch(new, kw.pop("lens", lens), **{**dict(max_len=128), **kw}), P.to_gpu(k), P.to_gpu(v))
        assert pool.cache.faults() == hip.KV_FAULT_BATCH, kw
    assert torch.equal(before.view(torch.int16), whole().view(torch.int16))


def test_streams_and_graphs(hip):
    """A call captured on another stream and replayed over changed contents, between eager work."""
    import torch

    rng = np.random.default_rng(4)
    nkv, hd, n = 2, 128, 5
    lens = [70, 1, 130, 64, 12]
    cap = [200] * n
    pool = P.Pool(hip, cap, nkv, hd, 64, "mxfp8")
    k, v = (P.to_gpu(_rows(rng, n, nkv, hd)) for _ in range(2))
    back = [torch.empty_like(k) for _ in range(2)]
    batch = pool.batch([1] * n, lens, max_len=200)
    side = torch.cuda.Stream()
    pool.cache.set_stream(side.cuda_stream)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pool.cache.append(0, batch, k, v)
        pool.cache.read(0, batch, *back)
    for step in range(4):
        x = _rows(rng, n, nkv, hd)
        k.copy_(P.to_gpu(x))
        v.copy_(P.to_gpu(-x))
        batch.lens += 3 * step
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _same(P.to_cpu(back[0]), P.quantised(x, "mxfp8"))
        _same(P.to_cpu(back[1]), P.quantised(-x, "mxfp8"))
    pool.cache.set_stream(None)
    assert pool.cache.faults() == 0


def test_binding_refuses_wrong_tensors(hip):
    import torch

    pool = P.Pool(hip, [64], 2, 64, 64, "bf16")
    b = pool.batch([4], [4])
    z = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    ok = z(4, 2, 64)
    for k, v in ((z(4, 3, 64), ok), (ok, z(5, 2, 64)), (z(4, 2, 64, t=torch.float16), ok), (z(4, 2, 32), ok),
                 (z(4, 128), ok), (ok.cpu(), ok), (z(2, 4, 64).transpose(0, 1), ok), (z(4, 2, 64, t=torch.float32), ok)):
        with pytest.raises(hip.AosError):
            pool.cache.append(0, b, k, v)
        with pytest.raises(hip.AosError):
            pool.cache.read(0, b, k, v)
    with pytest.raises(hip.AosError):
        pool.cache.append(0, b, ok, ok, q=z(4, 4, 64))
    with pytest.raises(hip.AosError):
        pool.cache.append(0, b, ok, ok, k_bias=z(2, 64))
    with pytest.raises(hip.AosError):
        pool.cache.append(0, hip.KVBatch(b.starts, b.lens, b.pages, 4, 1000), ok, ok)
    with pytest.raises(hip.AosError):
        hip.KVBatch(b.starts, b.lens, b.pages.float(), 4, 4)
    with pytest.raises(hip.AosError):
        hip.KVBatch(b.starts, b.starts, b.pages, 4, 4)
    with pytest.raises(hip.AosError):
        pool.cache.set_rope(np.zeros((4, 16)), np.zeros((4, 16)))
    pool.cache.set_rope(np.ones((3, 32)), np.zeros((3, 32)))
    with pytest.raises(hip.AosError, match="rotary"):
        pool.cache.append(0, b, ok, ok)
    pool.cache.set_rope()
    pool.cache.append(0, b, ok, ok)
    assert pool.cache.faults() == 0


def test_a_new_cache_on_another_stream(hip):
    """The first append to a large cache, on a stream that does not wait for the null stream, is not undone by the pages'
    first zeros; the same with the rotary tables."""
    import torch

    rng = np.random.default_rng(4)
    nkv, hd, n = 8, 128, 200
    x = [P.bf16(rng.standard_normal((n, nkv, hd))) for _ in range(2)]
    k, v = map(P.to_gpu, x)
    back = [torch.zeros_like(k) for _ in range(2)]
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32).cuda()  # noqa: E731
    side = torch.cuda.Stream()
    pages = 8 * (1 << 30) // (2 * nkv * hd * 2 * 256)
    batch = hip.KVBatch(i32(0, n), i32(n), i32(pages - 1).view(1, 1), n, n)
    torch.cuda.synchronize()
    cache = hip.KVCache(1, nkv, hd, 256, pages, "bf16")
    cache.set_stream(side.cuda_stream)
    cache.append(0, batch, k, v)
    torch.cuda.synchronize()
    cache.read(0, batch, *back)
    torch.cuda.synchronize()
    assert all(np.array_equal(P.to_cpu(b), y) for b, y in zip(back, x))
    cache.set_rope(-np.ones((n, hd // 2), np.float32), np.zeros((n, hd // 2), np.float32))
    cache.append(0, batch, k, v)
    cache.read(0, batch, *back)
    torch.cuda.synchronize()
    assert np.array_equal(P.to_cpu(back[0]), -x[0]) and np.array_equal(P.to_cpu(back[1]), x[1])


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_there_and_back_again(hip, fmt):
    """Streams read out of a cache with rotary tables and written to other pages hold, and attend to, what they did."""
    import torch

    rng = np.random.default_rng(6)
    nh, nkv, hd, lens = 4, 2, 128, [70, 1, 200]
    T = sum(lens)
    pool = P.Pool(hip, lens, nkv, hd, 64, fmt)
    other = P.Pool(hip, lens, nkv, hd, 128, fmt, seed=1)
    cos, sin = (f(np.arange(200)[:, None] * 3.0 ** -np.arange(hd // 2)).astype(np.float32) for f in (np.cos, np.sin))
    for p in (pool, other):
        p.cache.set_rope(cos, sin)
    q, k, v = (P.to_gpu(_rows(rng, T, h, hd)) for h in (nh, nkv, nkv))
    turned = torch.empty_like(q)
    pool.cache.append(0, pool.batch(lens, lens), k, v, q=q, q_out=turned)
    held = [torch.empty_like(k) for _ in range(2)]
    pool.cache.read(0, pool.batch(lens, lens), *held)
    again, back = torch.empty_like(q), [torch.empty_like(k) for _ in range(2)]
    other.cache.append(0, other.batch(lens, lens), *held, q=turned, q_out=again, rotated=True)
    other.cache.read(0, other.batch(lens, lens), *back)
    assert torch.equal(turned.view(torch.int16), again.view(torch.int16))
    out = [torch.empty_like(q) for _ in range(2)]
    for p, o in zip((pool, other), out):
        p.cache.attention(0, p.batch(lens, lens), turned, o)
        assert p.cache.faults() == 0
    for a, b in zip((*held, out[0]), (*back, out[1])):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    pool.cache.append(0, pool.batch(lens, lens), k, v)  # (the next call rotates again)
    pool.cache.read(0, pool.batch(lens, lens), *back)
    assert torch.equal(held[0].view(torch.int16), back[0].view(torch.int16))


def _turned(hip, fails):
    """A cache whose tables negate the keys; what `fails` does to it is refused, and its calls are as before."""
    import torch

    hd, n = 256, 20
    pool = P.Pool(hip, [n], 1, hd, 64, "bf16")
    x = P.bf16(np.random.default_rng(0).standard_normal((n, 1, hd)))
    k, batch = P.to_gpu(x), pool.batch([n], [n])
    back = [torch.empty_like(k) for _ in range(2)]
    zeros = np.zeros((n, hd // 2), np.float32)
    pool.cache.set_rope(zeros - 1, zeros)
    with pytest.raises(hip.AosError, match="out of memory"):
        fails(pool.cache)
    pool.cache.append(0, batch, k, k)
    pool.cache.read(0, batch, *back)
    _same(P.to_cpu(back[0]), -x)
    _same(P.to_cpu(back[1]), x)
    assert pool.cache.faults() == 0


def test_a_cache_that_does_not_fit(hip):
    """Its failed allocation is no later call's error."""
    _turned(hip, lambda cache: hip.KVCache(1, 8, 128, 256, 2000000, "bf16"))


def test_tables_that_do_not_fit(hip):
    """The tables that were set stay."""
    def fails(cache):
        few = np.zeros((1, 128), np.float32)  # (not read: the allocation comes first)
        if hip.lib().aoship_kv_cache_set_rope(cache.h, few.ctypes.data, few.ctypes.data, 2 ** 31 - 1):
            raise hip.AosError(hip.last_error())

    _turned(hip, fails)
