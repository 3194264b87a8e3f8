"""Log probabilities of rows of logits on the GPU against float64, ids and ranks exactly; and of a model's prompt."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _plain(x, t, n):
    """float64 rows -> (logprob, rank, entropy, ids, tops); -1 and NaN as documented"""
    T, V = x.shape
    lp, rank, ent = np.full(T, np.nan), np.full(T, -1), np.full(T, np.nan)
    ids, tops = np.full((T, n), -1), np.full((T, n), np.nan)
    for r in range(T):
        m = x[r].max()
        if not np.isfinite(m):  # (a NaN, +infinity, or nothing above minus infinity)
            continue
        d = x[r] - m
        e = np.exp(d)
        z = np.log(e.sum())
        ent[r] = z - (e[e > 0] * d[e > 0]).sum() / e.sum()
        order = np.lexsort((np.arange(V), -x[r]))[:n]
        ids[r], tops[r] = order, d[order] - z
        if 0 <= t[r] < V:
            lp[r] = d[t[r]] - z
            rank[r] = (x[r] > x[r, t[r]]).sum() + (x[r, :t[r]] == x[r, t[r]]).sum()
    return lp, rank, ent, ids, tops


def _close(got, want, V):
    """A thread adds up to V / 256 terms, then 2 log2 steps join them: each addition is off by half a step, 2^-24 of the
    sum; an exponential by 2^-23 and its argument's three roundings, 3 2^-24 |d|, where the mean of e |d| / l is at most
    ln V + 1 <= 20; the logarithm and the last two subtractions by 2^-24 of their results each."""
    tol = 2.0 ** -24 * ((V / 256 + 30 + 3 * 20) * (1 + 0 * want) + 4 * np.abs(np.nan_to_num(want, neginf=0)))
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5])


def _run(hip, x, t, n, op=None):
    """x: a device tensor [T, V]"""
    import torch

    T = x.shape[0]
    op = op or hip.LogProbs()
    lp, ent = (torch.full((T,), 7.0, device="cuda") for _ in range(2))
    rank = torch.full((T,), 7, dtype=torch.int32, device="cuda")
    ids = torch.full((T, n), 7, dtype=torch.int32, device="cuda") if n else None
    tops = torch.full((T, n), 7.0, device="cuda") if n else None
    op(x, torch.from_numpy(np.asarray(t, np.int32)).cuda(), lp, ent, rank, ids, tops)
    torch.cuda.synchronize()
    f = lambda a: a.cpu().numpy().astype(np.float64)  # noqa: E731
    return f(lp), rank.cpu().numpy(), f(ent), (ids.cpu().numpy() if n else np.zeros((T, 0))), (f(tops) if n else np.zeros((T, 0)))


def _compare(hip, x, t, n, op=None):
    import torch

    got = _run(hip, x, t, n, op)
    want = _plain(x.double().cpu().numpy(), t, n)
    V = x.shape[1]
    _close(got[0], want[0], V)
    assert (got[1] == want[1]).all(), (got[1], want[1])
    # e |d| <= 2^k e: the entropy's own sum has the same terms, weighted: as far off again, times the largest |d| that
    # counts (below e^-d = 2^-24 / V a term is nothing)
    with np.errstate(invalid="ignore"):
        assert ((np.abs(got[2] - want[2]) <= 2.0 ** -24 * (V / 256 + 90) * (2 + 2 * want[2])) | (np.isnan(got[2]) & np.isnan(want[2]))).all()
    assert (got[3] == want[3]).all(), (np.argwhere(got[3] != want[3])[:5], got[3][got[3] != want[3]][:5])
    _close(got[4], want[4], V)
    again = _run(hip, x, t, n, op)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(got, again))
    torch.cuda.synchronize()


def _logits(T, V, kind, seed, spare=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 3.0 * torch.randn((T, V + spare), generator=g, device="cuda")
    x[torch.arange(T), torch.randint(0, V, (T,), generator=g, device="cuda")] += 9.0
    x = x if kind == "f32" else x.bfloat16()
    return x[:, spare // 2:spare // 2 + V]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("T,V,n,spare", [(1, 1, 1, 0), (3, 2, 2, 1), (5, 31, 5, 3), (2, 33, 32, 0), (300, 64, 32, 5),
                                         (7, 1000, 20, 1), (2, 4097, 3, 7), (1, 152064, 20, 0), (64, 20001, 20, 0),
                                         (13, 50257, 32, 0), (2100, 2500, 5, 2), (1, 1500001, 32, 1), (3, 9000, 0, 1)])
def test_sizes(hip, kind, T, V, n, spare):
    x = _logits(T, V, kind, V + T, spare)
    t = np.random.default_rng(T).integers(0, V, T)
    t[T // 2:] = x.float().argmax(1).cpu().numpy()[T // 2:]
    _compare(hip, x, t, n)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_orders_and_ties(hip, kind):
    """Equal logits, rising and falling ones, few values, large values in every place of one thread (which overflow the
    list of candidates), zeros of both signs."""
    import torch

    V, n = 40000, 32
    i = torch.arange(V, device="cuda")
    rows = [torch.zeros(V), i * 0.001, -i * 0.001, (i % 7).float(), (i * 7919 % V).float() * 0.01,
            torch.where(i // 4 % 256 == 5, 4.0 + (i % 97) * 0.01, -1.0), torch.where(i // 8 % 256 == 250, 5.0, 0.0),
            torch.where(i % 2 == 0, 0.0, -0.0), torch.where(i % 3 == 1, 1e30, -1e30), torch.where(i == V - 1, -3.0e38, -3.3e38),
            torch.where(i < 20, 1.0, float("-inf")), torch.where(i == 777, -50.0, float("-inf"))]
    x = torch.stack([r.float().cuda() for r in rows])
    x = x if kind == "f32" else x.bfloat16()
    for rep in (1, 300):  # rows in slices, rows whole
        big = x.repeat(rep, 1)
        t = np.random.default_rng(rep).integers(0, V, len(big))
        t[:len(rows)] = 0
        t[len(rows) - 1] = 777
        if rep == 1:
            _compare(hip, big, t, n)
            continue
        got = _run(hip, big, t, n)
        want = _plain(x.double().cpu().numpy(), t[:len(rows)], n)
        assert (got[3].reshape(rep, len(rows), n) == want[3][None]).all()
        for k in range(len(rows)):
            _close(got[2].reshape(rep, -1)[:, k], np.full(rep, want[2][k]), V * 4)


def test_rows_without_probabilities(hip):
    """NaN, +infinity, nothing above minus infinity; targets out of range, of probability zero; neighbours are served."""
    V = 5000
    x = _logits(9, V, "f32", 3)
    x[0, 17], x[1, 4999], x[2, 0] = float("nan"), float("inf"), float("nan")
    x[3] = float("-inf")
    x[4] = float("nan")
    x[5, 100:] = float("-inf")
    t = np.array([0, 4999, 3, 5, 6, 200, -1, V, 7])
    for n in (0, 8):
        _compare(hip, x, t, n)


def test_outputs_are_each_optional_and_nothing_else_is_written(hip):
    import torch

    x, t = _logits(6, 777, "f32", 1), np.arange(6)
    full = _run(hip, x, t, 4)
    op, tt = hip.LogProbs(), torch.arange(6, dtype=torch.int32, device="cuda")
    e = torch.full((8,), 7.0, device="cuda")
    op(x, entropy=e[1:7])
    r = torch.full((8,), 7, dtype=torch.int32, device="cuda")
    op(x, tt, rank=r[1:7])
    i = torch.full((8, 4), 7, dtype=torch.int32, device="cuda")
    op(x, top_ids=i[1:7])
    torch.cuda.synchronize()
    assert np.array_equal(e[1:7].cpu().numpy().astype(np.float64), full[2]) and (e[[0, 7]] == 7).all()
    assert np.array_equal(r[1:7].cpu().numpy(), full[1]) and (r[[0, 7]] == 7).all()
    assert np.array_equal(i[1:7].cpu().numpy(), full[3]) and (i[[0, 7]] == 7).all()


def test_refusals(hip):
    import torch

    op, x = hip.LogProbs(), torch.zeros((3, 50), device="cuda")
    t = torch.zeros(3, dtype=torch.int32, device="cuda")
    o = torch.zeros(3, device="cuda")
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.t()), dict(logits=x.cpu()), dict(targets=t.long()),
                dict(targets=t[:2]), dict(targets=t.cpu()), dict(targets=None), dict(logprob=o[:2]), dict(logprob=o.double()),
                dict(top_ids=torch.zeros((3, 33), dtype=torch.int32, device="cuda")),
                dict(top_ids=torch.zeros((3, 3), dtype=torch.int32, device="cuda"),
                     top_logprobs=torch.zeros((3, 4), device="cuda")),
                dict(top_logprobs=torch.zeros((3, 8), device="cuda")[:, :4])):
        args = dict(logits=x, targets=t, logprob=o)
        args.update(bad)
        with pytest.raises(hip.AosError):
            op(**args)


def test_captured_into_a_graph(hip):
    """Replayed several times over other logits, with eager calls and synchronizations between."""
    import torch

    op = hip.LogProbs()
    x = _logits(2, 60000, "f32", 1)
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = [torch.zeros(2, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"),
           torch.zeros((2, 7), dtype=torch.int32, device="cuda"), torch.zeros((2, 7), device="cuda")]
    s = torch.cuda.Stream()
    op.set_stream(s.cuda_stream)
    s.wait_stream(torch.cuda.current_stream())
    op(x, t, *out)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        op(x, t, *out)
    eager = hip.LogProbs()
    for seed in range(5):
        x.copy_(_logits(2, 60000, "f32", seed))
        t.fill_(seed * 1000)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = _run(hip, x, t.cpu().numpy(), 7, eager)
        for a, b in zip(out, (want[0], want[2], want[1], want[3], want[4])):
            assert np.array_equal(a.cpu().numpy().astype(np.float64), b)


def test_a_models_prompt(hip):
    """Model.score: the outputs of a 50-token prompt (two runs of the LM head) against forward()'s logits after each token,
    and the last token's logits and the cache as forward leaves them."""
    import torch

    import oracle  # noqa: F401 (the model's weights)
    from test_gpu_model import _device_model
    from test_oracle_model import rings, tiny_model

    cfg, w, lora, scales, rank = tiny_model()
    rng = np.random.default_rng(11)
    n = 50
    ids, rg = rng.integers(0, cfg["vocab"], n), rings(rng, n, len(scales))
    dm = _device_model(hip, cfg, w, lora, scales, rank, max_seq=64)
    d_ids = torch.from_numpy(np.asarray(ids, np.int32)).cuda()
    d_rings = torch.from_numpy(rg.view(np.uint8).copy()).cuda()
    V, k = cfg["vocab"], 6
    last = torch.zeros(V, device="cuda")
    # the same calls for both, so that the caches hold the same: 44 tokens, then 6 one by one
    want = []
    dm.forward(d_ids[:44], d_rings[:44 * 40], last)
    want.append(last.double().cpu().numpy())
    for i in range(44, n):
        dm.forward(d_ids[i:i + 1], d_rings[40 * i:40 * i + 40], last)
        want.append(last.double().cpu().numpy())
    dm.reset_cache()
    t = torch.from_numpy(np.append(ids[1:], -1).astype(np.int32)).cuda()
    lp, ent = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    rk = torch.zeros(n, dtype=torch.int32, device="cuda")
    top, tlp = torch.zeros((n, k), dtype=torch.int32, device="cuda"), torch.zeros((n, k), device="cuda")
    mine = torch.zeros(V, device="cuda")
    dm.score(d_ids[:44], d_rings[:44 * 40], t[:44], lp[:44], ent[:44], rk[:44], top[:44], tlp[:44], logits=mine)
    assert dm.cache_len() == 44
    assert np.array_equal(mine.double().cpu().numpy(), want[0])
    for i in range(44, n):
        dm.score(d_ids[i:i + 1], d_rings[40 * i:40 * i + 40], t[i:i + 1], lp[i:i + 1], ent[i:i + 1], rk[i:i + 1],
                 top[i:i + 1], tlp[i:i + 1])
    assert dm.cache_len() == n
    torch.cuda.synchronize()
    # one row's logits at a time and 32 rows' are float32 sums of the same products in another order: 2^-24 of sum |w x| a
    # step, measured in the logits' own size here by their spread
    for j, logits in enumerate(want):
        i = 43 + j
        p = _plain(logits[None], [int(t[i])], k)
        tol = 1e-3 * np.abs(logits).max()
        assert np.allclose(tlp[i].cpu().numpy(), p[4][0], atol=tol) and abs(float(ent[i]) - p[2][0]) <= tol
        if int(t[i]) >= 0:
            assert abs(float(lp[i]) - p[0][0]) <= tol
    # rows inside the 44 (in both runs of the head), against forward() on the prompt up to them: other row counts, other
    # kernels, whose activations are rounded to bfloat16 after other sums (2e-2 is what the model's own tests allow)
    for i in (0, 5, 31, 32, 42):
        dm.reset_cache()
        dm.forward(d_ids[:i + 1], d_rings[:40 * i + 40], last)
        p = _plain(last.double().cpu().numpy()[None], [int(t[i])], k)
        tol = 2e-2 * float(last.abs().max())
        assert abs(float(lp[i]) - p[0][0]) <= tol and abs(float(tlp[i, 0]) - p[4][0, 0]) <= tol
    dm.reset_cache()
    dm.forward(d_ids, d_rings, last)
    assert torch.isfinite(lp[:-1]).all() and torch.isnan(lp[-1]) and int(rk[-1]) == -1
    with pytest.raises(hip.AosError, match="full"):
        dm.score(d_ids, d_rings, None, entropy=ent)
    with pytest.raises(hip.AosError, match="targets"):
        dm.score(d_ids[:1], d_rings[:40], None, logprob=lp[:1])
