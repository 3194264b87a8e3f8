"""The paged cache's rotary positions, attention weights and eviction on the GPU: positions and moved rows exactly, weights
against float64 with bounds from the arithmetic, and a sequence's whole life with them."""
import numpy as np
import pytest

import kv_plain as P
from test_gpu_kv_cache import SHAPES, _rows, _same

pytestmark = pytest.mark.gpu


def _tables(n, hd, base=3.0):
    a = np.arange(n)[:, None] * base ** -np.arange(hd // 2)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def _i32(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()


def _f32(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()


# ---- rotary positions ------------------------------------------------------------------------


def _turned(x, cos, sin, at, axes, bias):
    """x [T, heads, hd] with pair i turned by row at[axes[i], t] of the tables"""
    pair = np.arange(x.shape[-1] // 2)
    c, s = cos[at[axes].T, pair], sin[at[axes].T, pair]
    return P.bf16(P.rotated(x.astype(np.float32) + (0 if bias is None else bias), c, s))


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("n_axes,weave", [(1, False), (3, False), (3, True), (4, True)])
def test_positions(hip, fmt, nh, nkv, hd, page, n_axes, weave):
    import torch

    rng = np.random.default_rng(hd + n_axes)
    past, new = [0, 5, 30, 0], [1, 0, 40, page + 3]
    lens, T = [a + b for a, b in zip(past, new)], sum(new)
    pool = P.Pool(hip, lens, nkv, hd, page, fmt)
    cos, sin = _tables(900, hd)
    pool.cache.set_rope(cos, sin)
    half = hd // 2
    axes = np.arange(half) % n_axes if weave else np.sort(np.arange(half) * n_axes // half)
    axes[-1] = n_axes - 1  # (as many axes in the smallest heads too)
    if n_axes > 1:
        pool.cache.set_rope_axes(axes)
    at = rng.integers(0, 900, (n_axes, T))
    at[:, 0], at[0, 1] = 0, 899
    q, k, v = _rows(rng, T, nh, hd), _rows(rng, T, nkv, hd), _rows(rng, T, nkv, hd)
    b = [rng.standard_normal((h, hd)).astype(np.float32) for h in (nh, nkv, nkv)]
    out, wide = torch.zeros((T, nh, hd), dtype=torch.bfloat16, device="cuda"), _i32(np.pad(at, ((0, 0), (0, 5)), constant_values=-9))
    pool.cache.append(0, pool.batch(new, lens), P.to_gpu(k), P.to_gpu(v), q=P.to_gpu(q), q_out=out, q_bias=_f32(b[0]),
                      k_bias=_f32(b[1]), v_bias=_f32(b[2]), positions=wide[:, :T] if n_axes > 1 else wide[0, :T])
    _same(P.to_cpu(out), _turned(q, cos, sin, at, axes, b[0]))
    back = [torch.empty((T, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pool.cache.read(0, pool.batch(new, lens), *back)
    _same(P.to_cpu(back[0]), P.quantised(_turned(k, cos, sin, at, axes, b[1]), fmt))
    _same(P.to_cpu(back[1]), P.quantised(P.bf16(v.astype(np.float32) + b[2]), fmt))
    assert pool.cache.faults() == 0


def test_positions_in_the_cache_are_the_plain_append(hip):
    """The same positions on all axes as the rows' places: what append does without them, bit for bit; a position outside the
    tables counts as 0 and is reported."""
    import torch

    rng = np.random.default_rng(0)
    lens, hd = [50, 9], 128
    cos, sin = _tables(64, hd)
    k, v, q = (P.to_gpu(_rows(rng, 59, h, hd)) for h in (2, 2, 4))
    got = []
    at = np.concatenate([np.arange(50), np.arange(9)])
    for mode in ("plain", "one", "same", "three", "outside"):
        pool = P.Pool(hip, lens, 2, hd, 64, "bf16")
        pool.cache.set_rope(cos, sin)
        pos = None
        if mode in ("one", "outside"):
            pos = _i32(np.where(at == 0, 64 if mode == "outside" else 0, at))
        elif mode != "plain":
            pool.cache.set_rope_axes(np.arange(hd // 2) % 3)
            pos = _i32(np.stack([at] * 3)) if mode == "three" else _i32(at).expand(3, 59)
        out = torch.zeros_like(q)
        pool.cache.append(0, pool.batch(lens, lens), k, v, q=q, q_out=out, positions=pos)
        back = [torch.empty_like(k) for _ in range(2)]
        pool.cache.read(0, pool.batch(lens, lens), *back)
        got.append(torch.cat([out.flatten(), back[0].flatten(), back[1].flatten()]).view(torch.int16))
        assert pool.cache.faults() == (hip.KV_FAULT_POSITION if mode == "outside" else 0)
        assert torch.equal(got[0], got[-1]), mode


def test_position_refusals(hip):
    import torch

    pool = P.Pool(hip, [4], 1, 64, 64, "bf16")
    k = torch.zeros((4, 1, 64), dtype=torch.bfloat16, device="cuda")
    b, at = pool.batch([4], [4]), torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    with pytest.raises(hip.AosError, match="tables"):
        pool.cache.append(0, b, k, k, positions=at[0])
    pool.cache.set_rope(*_tables(10, 64))
    for bad in (at, at[0, :3], at[0].long(), at[0].cpu(), at[0, 0]):
        with pytest.raises(hip.AosError):
            pool.cache.append(0, b, k, k, positions=bad)
    with pytest.raises(hip.AosError, match="rotated"):
        pool.cache.append(0, b, k, k, positions=at[0], rotated=True)
    pool.cache.append(0, b, k, k, positions=at[0])
    for bad in (np.zeros(31, int), np.full(32, 4), np.full(32, -1), np.zeros(32)):
        with pytest.raises(hip.AosError):
            pool.cache.set_rope_axes(bad)
    pool.cache.set_rope_axes(np.arange(32) % 2)
    with pytest.raises(hip.AosError):
        pool.cache.append(0, b, k, k, positions=at[0])
    pool.cache.append(0, b, k, k, positions=at)
    pool.cache.set_rope_axes(None)
    pool.cache.append(0, b, k, k, positions=at[0])


# ---- attention weights -----------------------------------------------------------------------


def _weights(q, k, scale, window, nkv):
    """float64 weights [nkv, L] of one sequence, q [n, nh, hd] its last rows, k [L, nkv, hd]"""
    n, nh, _ = q.shape
    L = k.shape[0]
    w = np.zeros((nkv, L))
    with np.errstate(all="ignore"):
        for t in range(n):
            p = L - n + t
            if p < 0:
                continue
            lo = max(0, p + 1 - window) if window else 0
            for h in range(nh):
                kv = h // (nh // nkv)
                s = k[lo:p + 1, kv] @ q[t, h]
                # scores are float32 (as documented): past its largest number they are infinite, whatever the scale
                s = np.where(np.abs(s) > 3.4028235e38, np.copysign(np.inf, s), s) * scale
                e = np.exp(s - s.max())
                w[kv, lo:p + 1] += e / e.sum()
    return w


def _tolerance(q, k, scale, w, prior):
    """Scores are float32 sums of exact products: (hd + 4) 2^-24 S each, S = scale sum |q| |k| (kv_plain.attention_bound),
    which changes a probability by at most 2.2 times that with its normaliser; exponentials, and sums of up to 2^17 terms in
    pieces of 2^10: 2^-13 in all; the prior's addition half a step."""
    fin = lambda x: np.where(np.isfinite(x), x, 0)  # noqa: E731
    S = abs(scale) * np.abs(fin(q)).sum(-1).max(initial=0.0) * np.abs(fin(k)).max(initial=0.0)
    return (2.2 * (q.shape[-1] + 4) * 2.0 ** -24 * S + 2.0 ** -13) * np.abs(w) + 2.0 ** -24 * np.abs(prior) + 1e-30


def _check_weigh(hip, fmt, nh, nkv, hd, page, new, lens, window=0, scale=None, small=True, seed=0, k_rows=None, q_rows=None,
                 prior=True, in_place=False, spread=1.0):
    import torch

    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    pool = P.Pool(hip, lens, nkv, hd, page, fmt, seed=seed)
    pool.cache.set_small_batches(small)
    total = sum(lens)
    k = P.bf16(rng.standard_normal((total, nkv, hd))) if k_rows is None else k_rows
    pool.cache.append(0, pool.batch(lens, lens), P.to_gpu(k), P.to_gpu(np.zeros_like(k)))
    T = sum(new)
    q = P.bf16(spread * rng.standard_normal((T, nh, hd))) if q_rows is None else q_rows
    wide = torch.zeros((T + 1, nh + 1, hd), dtype=torch.bfloat16, device="cuda")
    wide[:T, :nh] = P.to_gpu(q)
    n, L = len(lens), max(lens)
    before = rng.random((n, nkv, L + 7)).astype(np.float32)
    got = torch.full((n, nkv + 1, L + 7), 7.0, device="cuda")
    out = got[:, :nkv]
    p = _f32(before) if prior else None
    if in_place:
        out.copy_(p)
        p = out
    start = out.clone()
    batch = pool.batch(new, lens)
    pool.cache.weigh(0, batch, wide[:T, :nh], out, scale=scale, window=window, prior=p)
    first = out.clone()
    assert pool.cache.faults() == 0
    kq = P.quantised(k, fmt)
    at, row = np.cumsum([0] + list(lens)), np.cumsum([0] + list(new))
    for s in range(n):
        ks, qs = kq[at[s]:at[s + 1]], q[row[s]:row[s + 1]]
        w = _weights(qs, ks, scale, window, nkv)
        pr = before[s, :, :lens[s]].astype(np.float64) if prior else 0 * w
        want, tol = w + pr, _tolerance(qs, ks, scale, w, pr)
        g = first[s, :, :lens[s]].double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            bad = ~((np.abs(g - want) <= tol) | (np.isnan(g) & np.isnan(want)))
        assert not bad.any(), (s, int(bad.sum()), np.argwhere(bad)[:4].tolist(), g[bad][:4], want[bad][:4])
        assert torch.equal(first[s, :, lens[s]:], start[s, :, lens[s]:])
    assert (got[:, nkv] == 7).all()
    if in_place:
        out.copy_(start)
    else:
        out.fill_(3.0)
    pool.cache.weigh(0, batch, wide[:T, :nh], out, scale=scale, window=window, prior=p)
    for s in range(n):
        assert torch.equal(out[s, :, :lens[s]].view(torch.int32), first[s, :, :lens[s]].contiguous().view(torch.int32))
    return pool


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("small", [True, False])
def test_weights_of_single_tokens(hip, fmt, nh, nkv, hd, page, window, small):
    """A row each (and none, and one of a sequence of one), by either kernel"""
    _check_weigh(hip, fmt, nh, nkv, hd, page, [1, 1, 0, 1, 1, 1], [1, 64, 20, 65, 300, 129], window, small=small)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("window", [0, 50])
def test_weights_of_many_rows(hip, fmt, nh, nkv, hd, page, window):
    """Whole prompts, chunks, padding in front (more rows than positions), a sequence without rows or positions"""
    _check_weigh(hip, fmt, nh, nkv, hd, page, [70, 3, 0, 40, 0, 1], [70, 200, 33, 25, 0, 300], window, prior=False)


@pytest.mark.parametrize("nh,nkv,new", [(28, 4, 4), (32, 1, 1), (33, 1, 1), (16, 2, 4), (40, 1, 1)])
@pytest.mark.parametrize("small", [True, False])
def test_weights_at_the_border_of_few_rows(hip, nh, nkv, new, small):
    _check_weigh(hip, "bf16", nh, nkv, 64, 64, [new] * 3, [40, 1000, 257], small=small, in_place=True)


@pytest.mark.parametrize("fmt,nh,nkv,hd,new,lens,window", [
    ("bf16", 7, 1, 128, [1, 1], [9001, 4500], 0), ("mxfp8", 7, 1, 128, [2, 3], [5000, 1030], 2000),
    ("bf16", 14, 2, 64, [1500], [1500], 0), ("mxfp4", 3, 1, 128, [700, 30], [2700, 2000], 1111),
    ("bf16", 4, 1, 256, [333], [1500], 0), ("mxfp8", 2, 2, 80, [600, 599], [600, 700], 100)])
def test_weights_of_long_sequences(hip, fmt, nh, nkv, hd, new, lens, window):
    _check_weigh(hip, fmt, nh, nkv, hd, 128, new, lens, window, seed=5)


def test_weights_of_many_sequences(hip):
    """Enough blocks for pieces of several"""
    rng = np.random.default_rng(4)
    lens = rng.integers(1, 1500, 130).tolist()
    lens[7] = 9000
    _check_weigh(hip, "bf16", 2, 1, 64, 64, [1] * 130, lens, seed=6)
    lens = rng.integers(200, 3000, 300).tolist()
    _check_weigh(hip, "mxfp8", 1, 1, 64, 64, [1] * 300, lens, 900, seed=7)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 5.0, 1e-30])
@pytest.mark.parametrize("new", [1, 90])
def test_weights_at_any_scale(hip, scale, new):
    _check_weigh(hip, "bf16", 4, 2, 64, 64, [new, new], [90, 200], scale=scale)


@pytest.mark.parametrize("new", [2, 100])
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_weights_with_infinities_and_nans(hip, fmt, new):
    """NaN and infinite keys and queries reach the weights of rows that see them, and of no others"""
    rng = np.random.default_rng(8)
    lens, nkv, hd = [300, 300, 300, 300], 2, 64
    k = P.bf16(rng.standard_normal((1200, nkv, hd)))
    k[299, 0, 3] = np.nan  # seen by the last row only
    k[300 + 10, 1, 5] = np.inf
    k[600:900, 0] = P.bf16(np.full((300, hd), -3.0e38))  # scores that overflow
    q = P.bf16(rng.standard_normal((4 * new, 4, hd)))
    q[3 * new, 0, 1] = np.nan
    q[2 * new:3 * new, :2] = np.abs(q[2 * new:3 * new, :2]) + 1
    _check_weigh(hip, fmt, 4, nkv, hd, 64, [new] * 4, lens, k_rows=k, q_rows=q, small=new < 50)


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("hd,nkv,nh,new,window", [(128, 8, 24, 1, 0), (128, 8, 24, 20, 700), (256, 2, 16, 1, 0), (64, 4, 28, 45, 0)])
def test_weights_with_the_chip_full(hip, fmt, hd, nkv, nh, new, window):
    """More workgroups than the chip holds, converting and multiplying at once, against float64 sums over the values that the
    cache holds, and the same bits three times."""
    import torch

    rng = np.random.default_rng(hd + new)
    lens = rng.integers(new, 3000, 64).tolist()
    pool = P.Pool(hip, lens, nkv, hd, 128, fmt)
    total, T, g = sum(lens), 64 * new, nh // nkv
    gen = torch.Generator(device="cuda").manual_seed(hd)
    k = torch.randn((total, nkv, hd), generator=gen, device="cuda").bfloat16()
    pool.cache.append(0, pool.batch(lens, lens), k, k)
    held = [torch.empty_like(k) for _ in range(2)]
    pool.cache.read(0, pool.batch(lens, lens), *held)
    q = torch.randn((T, nh, hd), generator=gen, device="cuda").bfloat16()
    out = torch.zeros((64, nkv, max(lens)), device="cuda")
    b = pool.batch([new] * 64, lens)
    pool.cache.weigh(0, b, q, out, window=window)
    first = out.clone()
    S = hd ** -0.5 * float(q.float().abs().sum(-1).max()) * float(held[0].float().abs().max())
    rel = 2.2 * (hd + 4) * 2.0 ** -24 * S + 2.0 ** -13  # (_tolerance)
    at = 0
    for s, L in enumerate(lens):
        x = held[0][at:at + L].double().permute(1, 2, 0).contiguous()
        at += L
        y = q[s * new:(s + 1) * new].double().unflatten(1, (nkv, g)).permute(1, 0, 2, 3).reshape(nkv, new * g, hd)
        far = (L - new + torch.arange(new, device="cuda"))[:, None] - torch.arange(L, device="cuda")
        hidden = (far < 0) | (far >= window) if window else far < 0
        z = torch.matmul(y, x) * hd ** -0.5
        z = z.masked_fill(hidden.repeat_interleave(g, 0), float("-inf"))
        want = torch.softmax(z, -1).sum(1)
        got = first[s, :, :L].double()
        assert ((got - want).abs() <= rel * want + 1e-30).all(), (s, float(((got - want).abs() / (want + 1e-30)).max()))
    for _ in range(2):
        out.zero_()
        pool.cache.weigh(0, b, q, out, window=window)
        assert torch.equal(out, first)


def _state(pool, n, nkv, L):
    import torch

    return torch.full((n, nkv, L), 7.0, device="cuda")


@pytest.mark.parametrize("new", [1, 60])
def test_weights_and_bad_batches(hip, new):
    """Bad pages are left out of the sums and keep their prior; sequences that do not fit are left out; others are served."""
    import torch

    rng = np.random.default_rng(3)
    lens, nkv, hd, nh = [300, 200, 100], 2, 64, 6
    pool = P.Pool(hip, lens, nkv, hd, 64, "bf16")
    k = P.bf16(rng.standard_normal((600, nkv, hd)))
    pool.cache.append(0, pool.batch(lens, lens), P.to_gpu(k), P.to_gpu(k))
    q = P.bf16(rng.standard_normal((3 * new, nh, hd)))
    pool.pages[0, 1] = 10 ** 6
    pool.pages[2, 0] = -1
    out = _state(pool, 3, nkv, 300)
    pool.cache.weigh(0, pool.batch([new] * 3, lens), P.to_gpu(q), out, scale=0.125)
    assert pool.cache.faults() == hip.KV_FAULT_PAGE
    seen = k[:300].copy()
    w = np.zeros((nkv, 300))
    for t in range(new):
        for h in range(nh):
            s = np.where((np.arange(300) <= 300 - new + t) & (np.arange(300) // 64 != 1), seen[:, h // 3] @ q[t, h] * 0.125, -np.inf)
            e = np.exp(s - s.max())
            w[h // 3] += e / e.sum()
    got = out.double().cpu().numpy()
    assert np.allclose(got[0], w, rtol=1e-3, atol=1e-6) and (got[0, :, 64:128] == 0).all()
    assert np.allclose(got[1, :, :200], _weights(q[new:2 * new], k[300:500], 0.125, 0, nkv), rtol=1e-3, atol=1e-6)
    assert (got[2, :, :64] == 0).all() and (got[1, :, 200:] == 7).all()
    # lengths and rows that do not fit
    out = _state(pool, 3, nkv, 300)
    pool.cache.weigh(0, pool.batch([new] * 3, [301, 200, -1], max_len=300), P.to_gpu(q), out)
    assert pool.cache.faults() & hip.KV_FAULT_BATCH
    got = out.cpu().numpy()
    assert (got[0] == 7).all() and (got[2] == 7).all() and (got[1, :, :200] != 7).all()
    out = _state(pool, 3, nkv, 300)
    pool.cache.weigh(0, pool.batch([new] * 3, lens, starts=[0, 2 * new, new, 3 * new], max_new=2 * new), P.to_gpu(q), out)
    assert pool.cache.faults() & hip.KV_FAULT_BATCH
    torch.cuda.synchronize()


@pytest.mark.parametrize("new,window", [(1, 0), (40, 64)])
def test_weights_captured_into_a_graph(hip, new, window):
    """Replayed with other queries, lengths and pages within the bounds, eager calls between; a call that needs more
    workspace than was reserved is refused while the stream is captured."""
    import torch

    rng = np.random.default_rng(1)
    lens, nkv, hd, nh, L = [200, 400], 2, 64, 6, 512
    pool = P.Pool(hip, [512, 512], nkv, hd, 64, "bf16")
    k = P.to_gpu(P.bf16(rng.standard_normal((1024, nkv, hd))))
    pool.cache.append(0, pool.batch([512] * 2, [512] * 2), k, k)
    b = pool.batch([new] * 2, lens, max_len=L)
    q = P.to_gpu(P.bf16(rng.standard_normal((2 * new, nh, hd))))
    out, prior = torch.zeros((2, nkv, L), device="cuda"), torch.rand((2, nkv, L), device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    pool.cache.set_stream(s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(hip.AosError, match="reserve"):
        with torch.cuda.graph(g, stream=s):
            pool.cache.weigh(0, b, q, out, window=window, prior=prior)
    torch.cuda.synchronize()
    pool.cache.reserve_weigh(nh, b, 2 * new)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pool.cache.weigh(0, b, q, out, window=window, prior=prior)
    eager = torch.zeros_like(out)
    for i in range(5):
        b.lens.copy_(_i32(rng.integers(new, L + 1, 2)))
        q.copy_(P.to_gpu(P.bf16(rng.standard_normal((2 * new, nh, hd)))))
        torch.cuda.synchronize()
        out.zero_()
        eager.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        pool.cache.weigh(0, b, q, eager, window=window, prior=prior)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and float(out.sum()) > 0


# ---- eviction --------------------------------------------------------------------------------


def _chosen(w, L, keep, first, recent):
    """kept positions of one head"""
    n = min(keep, L)
    if n == L:
        return np.arange(L)
    mid = np.arange(first, L - recent)
    x = np.where(np.isnan(w[mid]), -np.inf, w[mid]) + 0.0
    nan = np.isnan(w[mid])
    best = mid[np.lexsort((mid, nan, -x))][:n - first - recent]
    return np.sort(np.concatenate([np.arange(first), np.arange(L - recent, L), best]))


def _evicted(hip, fmt, nkv, hd, page, lens, keep, first, recent, weights, layers=1, seed=0):
    """Runs an eviction and checks everything it writes and what it must not."""
    import torch

    rng = np.random.default_rng(seed)
    weights = np.asarray(weights, np.float32)  # (as the call gets them)
    kept = [min(a, b) for a, b in zip(keep, lens)]
    pages = lambda n: -(-n // page)  # noqa: E731
    pool = P.Pool(hip, lens, nkv, hd, page, fmt, layers=layers, spare=sum(map(pages, kept)) + 3, seed=seed)
    total = sum(lens)
    k, v = (P.bf16(rng.standard_normal((total, nkv, hd)) * np.exp2(rng.integers(-3, 4, (total, nkv, 1)))) for _ in range(2))
    layer = layers - 1
    whole = pool.batch(lens, lens)
    pool.cache.append(layer, whole, P.to_gpu(k), P.to_gpu(v))
    to, at = np.full((len(lens), max(map(pages, kept)) + 1), -1, np.int32), 0
    for s, n in enumerate(kept):
        to[s, :pages(n)] = pool.spare[at:at + pages(n)]
        at += pages(n)
    most, L = max(kept), max(lens)
    out = torch.full((len(lens), nkv, most + 3), -7, dtype=torch.int32, device="cuda")
    wo = torch.full((len(lens), nkv, L + 2), 7.0, device="cuda")
    w = _f32(weights)
    before = [torch.empty((total, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pool.cache.read(layer, whole, *before)
    pool.cache.evict(layer, whole, w, _i32(keep), _i32(to), out, first=first, recent=recent, weights_out=wo)
    assert pool.cache.faults() == 0
    got, gw = out.cpu().numpy(), wo.cpu().numpy()
    T = sum(kept)
    rows = [np.zeros((T, nkv, hd)) for _ in range(2)]
    r0 = p0 = 0
    kq, vq = P.quantised(k, fmt), P.quantised(v, fmt)
    for s in range(len(lens)):
        for h in range(nkv):
            want = _chosen(weights[s, h], lens[s], keep[s], first, recent)
            assert np.array_equal(got[s, h, :kept[s]], want), (s, h, got[s, h, :kept[s]][:20], want[:20])
            rows[0][r0:r0 + kept[s], h], rows[1][r0:r0 + kept[s], h] = kq[p0 + want, h], vq[p0 + want, h]
            assert np.array_equal(gw[s, h, :kept[s]], weights[s, h, want].astype(np.float32), equal_nan=True)
        assert (got[s, :, kept[s]:] == -7).all()
        assert (gw[s, :, kept[s]:lens[s]] == 0).all() and (gw[s, :, lens[s]:] == 7).all()
        r0 += kept[s]
        p0 += lens[s]
    if T:
        b = hip.KVBatch(_i32(np.cumsum([0] + kept)), _i32(kept), _i32(to), most, most)
        back = [torch.empty((T, nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        pool.cache.read(layer, b, *back)
        _same(P.to_cpu(back[0]), rows[0])
        _same(P.to_cpu(back[1]), rows[1])
    after = [torch.empty_like(x) for x in before]
    pool.cache.read(layer, whole, *after)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(before, after))
    if layers > 1:
        pool.cache.read(0, pool.batch(lens, lens), *after)
        assert all((a == 0).all() for a in after)
    assert pool.cache.faults() == 0
    return pool, to, kept


@pytest.mark.parametrize("fmt", P.FORMATS)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
def test_evict(hip, fmt, nh, nkv, hd, page):
    """Kept counts at and off tile and unit borders, of everything, of nothing; ragged lengths"""
    rng = np.random.default_rng(nh)
    lens = [300, 1, 64, 200, 500, 130, 0]
    keep = [128, 5, 64, 77, 257, 9, 3]
    w = rng.random((7, nkv, 500)) ** 4
    w[rng.random(w.shape) < 0.3] = 0.0
    _evicted(hip, fmt, nkv, hd, page, lens, keep, 2, 6, w, layers=2)


def test_evict_orders(hip):
    """Equal weights, rising and falling ones, infinities, NaNs, negative ones, zeros of both signs"""
    rng = np.random.default_rng(0)
    L, nkv = 3000, 2
    rows = [np.zeros(L), np.arange(L), -np.arange(L), np.full(L, np.nan), np.arange(L) % 3, np.full(L, -np.inf), rng.random(L),
            np.where(rng.random(L) < 0.5, np.nan, rng.random(L)), np.where(np.arange(L) % 2, 0.0, -0.0),
            np.where(rng.random(L) < 0.9, np.inf, 1.0), np.where(np.arange(L) == 1500, 1.0, 0.0), rng.random(L) * 1e-42]
    w = np.stack([np.stack([r, r[::-1]]) for r in rows])
    n = len(rows)
    for keep, first, recent in ((1000, 0, 0), (1, 0, 0), (100, 40, 60), (2999, 1, 1), (64, 0, 63), (0, 0, 0)):
        _evicted(hip, "bf16", nkv, 64, 64, [L] * n, [keep] * n, first, recent, w)


@pytest.mark.parametrize("L", [32767, 32768, 32769, 70001])
def test_evict_of_long_sequences(hip, L):
    """More weights than a workgroup holds; ties across its spans"""
    rng = np.random.default_rng(L)
    w = np.floor(rng.random((2, 1, L)) ** 3 * 50)
    w[1] = rng.random((1, L))
    _evicted(hip, "mxfp4", 1, 64, 256, [L, L - 1000], [L // 3, L // 2], 4, 100, w)


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_evict_and_bad_batches(hip, fmt):
    """Sequences that do not fit are left out, positions of bad pages move as zeros and not to bad pages, others are served."""
    import torch

    rng = np.random.default_rng(2)
    nkv, hd, L = 2, 64, 200
    lens = [200, 200, 200, 201, 200]
    pool = P.Pool(hip, [200] * 5, nkv, hd, 64, fmt, spare=20)
    rows = P.bf16(rng.standard_normal((1000, nkv, hd)) + 5)
    pool.cache.append(0, pool.batch([200] * 5, [200] * 5), P.to_gpu(rows), P.to_gpu(rows))
    pool.pages[0, 1] = 999
    to = np.concatenate([pool.spare, [0] * 10])[:20].reshape(5, 4).astype(np.int32)[:, :2]
    to[4, 1] = -5
    keep = [100, -1, 9, 100, 100]  # (9: less than first + recent)
    w = np.zeros((5, nkv, L), np.float32)
    w[:, :, 50:180] = 1
    kept = torch.full((5, nkv, 100), -7, dtype=torch.int32, device="cuda")
    wo = torch.full((5, nkv, L), 7.0, device="cuda")
    pool.cache.evict(0, pool.batch([200] * 5, lens, max_len=200), _f32(w), _i32(keep), _i32(to), kept, first=4, recent=6, weights_out=wo)
    assert pool.cache.faults() == hip.KV_FAULT_PAGE | hip.KV_FAULT_BATCH
    got = kept.cpu().numpy()
    want = _chosen(w[0, 0], 200, 100, 4, 6)
    assert (got[[0, 0, 4, 4], [0, 1, 0, 1]] == want).all()
    for s in (1, 2, 3):
        assert (got[s] == -7).all() and (wo[s] == 7).all()
    back = [torch.full((64, nkv, hd), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for s in (0, 4):
        b = hip.KVBatch(_i32([0, 64]), _i32([64]), _i32(to[s:s + 1, :1]), 64, 64)
        pool.cache.read(0, b, *back)
        x = P.quantised(rows, fmt)[200 * s + want[:64]]
        if s == 0:
            x[(want[:64] >= 64) & (want[:64] < 128)] = 0
        _same(P.to_cpu(back[0]), x)
        _same(P.to_cpu(back[1]), x)
    assert pool.cache.faults() == 0


def test_evict_refusals(hip):
    import torch

    pool = P.Pool(hip, [100, 100], 2, 64, 64, "bf16")
    b = pool.batch([1, 1], [100, 100])
    w, i = torch.zeros((2, 2, 100), device="cuda"), torch.zeros((2, 2, 100), dtype=torch.int32, device="cuda")
    good = dict(weights=w, keep=i[:, 0, 0].contiguous(), to_pages=i[:, 0, :2].contiguous(), kept=i.clone())
    pool.cache.evict(0, b, **good)
    for bad in (dict(weights=w[:, :, :99]), dict(weights=w.double()), dict(weights=w[:1]), dict(weights=w.cpu()),
                dict(weights=w.transpose(1, 2)), dict(keep=good["keep"].long()), dict(keep=good["keep"][:1]), dict(kept=w),
                dict(kept=i[:, :1]), dict(to_pages=good["to_pages"].long()), dict(to_pages=good["to_pages"][:1]),
                dict(weights_out=w), dict(weights_out=w[:, :, :50]), dict(first=-1), dict(recent=-1)):
        with pytest.raises(hip.AosError):
            pool.cache.evict(0, b, **{**good, **bad})
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (dict(weights=w[:, :, :99]), dict(weights=w.double()), dict(prior=w[:, :, :99]), dict(window=-1), dict(q=q[:, :3]),
                dict(scale=float("inf"))):
        with pytest.raises(hip.AosError):
            pool.cache.weigh(0, b, **{**dict(q=q, weights=w), **bad})
    for bad in ((3, 1), (4, 0)):
        with pytest.raises(hip.AosError):
            pool.cache.reserve_weigh(bad[0], b, bad[1])


def test_evict_captured_into_a_graph(hip):
    import torch

    rng = np.random.default_rng(9)
    nkv, hd, L = 2, 64, 300
    pool = P.Pool(hip, [L, L], nkv, hd, 64, "mxfp8", spare=8)
    rows = P.to_gpu(_rows(rng, 2 * L, nkv, hd))
    pool.cache.append(0, pool.batch([L] * 2, [L] * 2), rows, rows)
    b, to = pool.batch([L] * 2, [L] * 2), _i32(pool.spare[:8].reshape(2, 4))
    w, keep = torch.zeros((2, nkv, L), device="cuda"), _i32([100, 200])
    kept, wo = torch.zeros((2, nkv, 250), dtype=torch.int32, device="cuda"), torch.zeros((2, nkv, L), device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    pool.cache.set_stream(s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pool.cache.evict(0, b, w, keep, to, kept, first=4, recent=8, weights_out=wo)
    for i in range(4):
        lens, n = rng.integers(150, L + 1, 2), rng.integers(20, 250, 2)
        x = rng.random((2, nkv, L)).astype(np.float32)
        w.copy_(_f32(x))
        keep.copy_(_i32(n))
        b.lens.copy_(_i32(lens))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for q in range(2):
            for h in range(nkv):
                want = _chosen(x[q, h], lens[q], n[q], 4, 8)
                assert np.array_equal(kept[q, h, :len(want)].cpu().numpy(), want)
                assert np.array_equal(wo[q, h, :len(want)].cpu().numpy(), x[q, h, want])
    assert pool.cache.faults() == 0


# ---- all of them together --------------------------------------------------------------------


@pytest.mark.parametrize("fmt", P.FORMATS)
def test_a_sequences_life(hip, fmt):
    """Two layers, two sequences: prompts with image positions are appended and attended to, the weights of their last rows
    choose what stays, the rest is evicted, and decoding goes on at the texts' own positions; every attention and weight
    against float64 over the rows that each head kept."""
    import torch

    rng = np.random.default_rng(12)
    nh, nkv, hd, page, layers = 6, 2, 64, 64, 2
    lens, keep, first, recent, look = [150, 90], [70, 64], 3, 20, 16
    cos, sin = _tables(400, hd, 1.7)
    axes = np.arange(hd // 2) % 3
    pool = P.Pool(hip, [256, 256], nkv, hd, page, fmt, layers=layers, spare=6)
    cache = pool.cache
    cache.set_rope(cos, sin)
    cache.set_rope_axes(axes)
    T = sum(lens)
    at = rng.integers(0, 200, (3, T))
    to = _i32(np.pad(pool.spare[:6].reshape(2, 3), ((0, 0), (0, 2)), constant_values=-1))
    kv, acc, kept = [], [], []
    for layer in range(layers):
        q, k, v = (_rows(rng, T, h, hd) for h in (nh, nkv, nkv))
        gq = P.to_gpu(q)
        cache.append(layer, pool.batch(lens, lens), P.to_gpu(k), P.to_gpu(v), q=gq, q_out=gq, positions=_i32(at))
        out = torch.empty_like(gq)
        cache.attention(layer, pool.batch(lens, lens), gq, out)
        qr, kr, vr = P.to_cpu(gq), P.quantised(_turned(k, cos, sin, at, axes, None), fmt), P.quantised(v, fmt)
        tail = np.concatenate([np.arange(o + n - look, o + n) for o, n in ((0, 150), (150, 90))])
        w = torch.zeros((2, nkv, 256), device="cuda")
        cache.weigh(layer, pool.batch([look] * 2, lens), gq[torch.from_numpy(tail).cuda()].contiguous(), w)
        state = torch.zeros((2, nkv, 256), device="cuda")
        pos = torch.full((2, nkv, 70), -1, dtype=torch.int32, device="cuda")
        cache.evict(layer, pool.batch([look] * 2, lens), w, _i32(keep), to, pos, first=first, recent=recent, weights_out=state)
        heads = []
        for s, (o, n) in enumerate(((0, 150), (150, 90))):
            a, bnd = P.attention(qr[o:o + n], kr[o:o + n], vr[o:o + n], hd ** -0.5)
            tol = P.attention_bound(qr[o:o + n], kr[o:o + n], bnd, a, hd ** -0.5)
            assert (np.abs(P.to_cpu(out[o:o + n]) - a) <= tol).all()
            want = _weights(qr[o + n - look:o + n], kr[o:o + n], hd ** -0.5, 0, nkv)
            got = w[s, :, :n].double().cpu().numpy()
            assert (np.abs(got - want) <= _tolerance(qr[o + n - look:o + n], kr[o:o + n], hd ** -0.5, want, 0)).all()
            mine = [_chosen(got[h], n, keep[s], first, recent) for h in range(nkv)]
            assert all(np.array_equal(pos[s, h, :keep[s]].cpu().numpy(), mine[h]) for h in range(nkv))
            heads.append([np.stack([x[o:o + n][mine[h], h] for h in range(nkv)], 1) for x in (kr, vr)])
        kv.append(heads)
        acc.append(state)
    assert cache.faults() == 0
    # decoding goes on: ten tokens each, at the positions that follow the texts
    for step in range(10):
        lens_now = [n + step + 1 for n in keep]
        b = hip.KVBatch(_i32([0, 1, 2]), _i32(lens_now), to, 1, 256)
        where = np.stack([np.full(3, 150 + step), np.full(3, 90 + step)], 1)
        for layer in range(layers):
            q, k, v = (_rows(rng, 2, h, hd) for h in (nh, nkv, nkv))
            gq = P.to_gpu(q)
            cache.append(layer, b, P.to_gpu(k), P.to_gpu(v), q=gq, q_out=gq, positions=_i32(where))
            out = torch.empty_like(gq)
            cache.attention(layer, b, gq, out)
            before = acc[layer].clone()
            cache.weigh(layer, b, gq, acc[layer], prior=acc[layer])
            qr, kr, vr = P.to_cpu(gq), P.quantised(_turned(k, cos, sin, where, axes, None), fmt), P.quantised(v, fmt)
            for s in range(2):
                h = kv[layer][s]
                h[0], h[1] = np.concatenate([h[0], kr[s:s + 1]]), np.concatenate([h[1], vr[s:s + 1]])
                a, bnd = P.attention(qr[s:s + 1], h[0], h[1], hd ** -0.5)
                assert (np.abs(P.to_cpu(out[s:s + 1]) - a) <= P.attention_bound(qr[s:s + 1], h[0], bnd, a, hd ** -0.5)).all()
                want, pr = _weights(qr[s:s + 1], h[0], hd ** -0.5, 0, nkv), before[s, :, :lens_now[s]].double().cpu().numpy()
                got = acc[layer][s, :, :lens_now[s]].double().cpu().numpy()
                assert (np.abs(got - pr - want) <= _tolerance(qr[s:s + 1], h[0], hd ** -0.5, want, pr)).all()
    assert cache.faults() == 0


# ---- attention weights of batches whose sequences differ much ----------------------------------


@pytest.mark.parametrize("fmt,nh,nkv,hd,window", [("bf16", 28, 4, 128, 0), ("mxfp8", 24, 8, 128, 300), ("mxfp4", 14, 2, 64, 0),
                                                  ("bf16", 4, 1, 256, 100)])
@pytest.mark.parametrize("place", ["first", "last", "middle"])
def test_weights_of_one_prompt_beside_single_tokens(hip, fmt, nh, nkv, hd, window, place):
    """What a serving step has: a prompt's chunk and many streams of a token each, some of none"""
    new, lens = [1, 0, 1] * 24, [5 + 17 * i for i in range(72)]
    at = {"first": 0, "last": 72, "middle": 31}[place]
    new.insert(at, 260)
    lens.insert(at, 700)
    _check_weigh(hip, fmt, nh, nkv, hd, 64, new, lens, window, seed=at)


def test_weights_of_ragged_prompts(hip):
    """More sequences than one step of the search for a row's sequence takes, rows in front of the first one's and behind
    the last one's, and a workspace for batches of any spread"""
    import torch

    rng = np.random.default_rng(2)
    n, nkv, nh, hd = 150, 1, 3, 64
    new = np.where(rng.random(n) < 0.8, rng.integers(0, 3, n), rng.integers(3, 200, n))
    lens = (new + rng.integers(0, 100, n)).tolist()
    _check_weigh(hip, "bf16", nh, nkv, hd, 64, new.tolist(), lens, seed=3)
    pool = P.Pool(hip, lens, nkv, hd, 64, "bf16")
    k = P.to_gpu(P.bf16(rng.standard_normal((sum(lens), nkv, hd))))
    pool.cache.append(0, pool.batch(lens, lens), k, k)
    starts = np.concatenate([[0], np.cumsum(new)])
    T = int(starts[-1])
    q = torch.zeros((T + 60, nh, hd), dtype=torch.bfloat16, device="cuda")
    q[40:40 + T] = P.to_gpu(P.bf16(rng.standard_normal((T, nh, hd))))
    got = [torch.full((n, nkv, max(lens)), 7.0, device="cuda") for _ in range(2)]
    pool.cache.weigh(0, pool.batch(new, lens), q[40:40 + T], got[0])
    pool.cache.weigh(0, pool.batch(new, lens, starts=starts + 40), q, got[1])
    assert torch.allclose(got[0], got[1], rtol=1e-5, atol=1e-7) and pool.cache.faults() == 0
    # starts that fall, sequences with rows before 0 and behind n_tokens: noted, and the rest within bounds
    for bad in (starts[::-1], np.where(np.arange(n + 1) == 70, 0, starts + 40)):
        pool.cache.weigh(0, pool.batch(new, lens, starts=bad), q, got[1])
        assert pool.cache.faults() & hip.KV_FAULT_BATCH
    out = torch.full((n, nkv, max(lens)), 7.0, device="cuda")
    pool.cache.weigh(0, pool.batch(new, lens, starts=starts - 5), q, out)
    assert pool.cache.faults() == hip.KV_FAULT_BATCH and (out[0] == 7).all() and (out[-1, 0, :lens[-1]] != 7).all()
    pool.cache.weigh(0, pool.batch(new, lens, starts=starts + 61), q, out)
    assert pool.cache.faults() == hip.KV_FAULT_BATCH


@pytest.mark.parametrize("new", [1, 40])
def test_a_graph_keeps_its_workspace(hip, new):
    """Eager calls and a second graph that need a larger one, between the replays of a graph captured before"""
    import torch

    rng = np.random.default_rng(new)
    lens, nkv, hd, nh = [200, 400], 2, 64, 6
    pool = P.Pool(hip, [2048, 2048], nkv, hd, 64, "bf16")
    k = P.to_gpu(P.bf16(rng.standard_normal((4096, nkv, hd))))
    pool.cache.append(0, pool.batch([2048] * 2, [2048] * 2), k, k)
    small, large = pool.batch([new] * 2, lens), pool.batch([300, 200], [2048, 1900])
    q = [P.to_gpu(P.bf16(rng.standard_normal((n, nh, hd)))) for n in (2 * new, 500)]
    out = [torch.zeros((2, nkv, n), device="cuda") for n in (400, 2048)]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    pool.cache.set_stream(s.cuda_stream)
    pool.cache.reserve_weigh(nh, small, 2 * new)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0], stream=s):
        pool.cache.weigh(0, small, q[0], out[0])
    free = torch.cuda.mem_get_info()[0]
    pool.cache.weigh(0, large, q[1], out[1])
    torch.cuda.synchronize()
    want = [torch.zeros_like(out[0]), out[1].clone()]
    assert torch.cuda.mem_get_info()[0] < free
    with torch.cuda.graph(graphs[1], stream=s):
        pool.cache.weigh(0, large, q[1], out[1])
    pool.cache.weigh(0, small, q[0], want[0])
    torch.cuda.synchronize()
    for i in range(3):
        filler = torch.full((1 << 22,), 5.0, device="cuda")  # (as what would be freed might be used again)
        for g, o, w in zip(graphs, out, want):
            o.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, w) and float(o.sum()) > 0
        assert (filler == 5).all()
        del filler


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("e", [10, 20, 29])
def test_weights_of_large_scores(hip, new, e):
    """Scores of up to 2^30, as documented, exact in float32 (one product each) and hundreds apart or equal: a row's weight
    goes to its largest ones alike. 100 equal terms are added (half a step each, 2^-24), an exponential and an inverse
    taken, and 120 rows added up: 2^-16 of a weight in all."""
    import torch

    lens, nkv, nh, hd = [300, 65], 2, 4, 64
    k = np.zeros((sum(lens), nkv, hd))
    for o, n in ((0, 300), (300, 65)):
        k[o:o + n:3, :, 0], k[o + 1:o + n:3, :, 0] = 2.0 ** e * 1.171875, 2.0 ** (e - 1)
    q = np.zeros((2 * new, nh, hd))
    q[..., 0] = 1.6875  # (products of up to 1.98 2^e)
    q[::2, 1, 0] = -1.6875
    pool = P.Pool(hip, lens, nkv, hd, 64, "bf16")
    pool.cache.append(0, pool.batch(lens, lens), P.to_gpu(k), P.to_gpu(k))
    out = torch.full((2, nkv, 300), 7.0, device="cuda")
    pool.cache.weigh(0, pool.batch([new] * 2, lens), P.to_gpu(q), out, scale=1.0)
    got = out.double().cpu().numpy()
    for s, (o, n) in enumerate(((0, 300), (300, 65))):
        want = _weights(q[s * new:(s + 1) * new], k[o:o + n], 1.0, 0, nkv)
        assert want.max() > 0.003 and (np.abs(got[s, :, :n] - want) <= 2.0 ** -16 * want + 1e-30).all()


def test_weights_of_thousands_of_sequences(hip):
    """A row's sequence searched for in three steps"""
    rng = np.random.default_rng(4)
    n = 5000
    new = (rng.random(n) < 0.5).astype(int)
    lens = new + rng.integers(0, 4, n)
    new[4321], lens[4321] = 300, 333
    new[77], lens[77] = 40, 40
    _check_weigh(hip, "bf16", 2, 1, 64, 64, new.tolist(), lens.tolist(), seed=9)
