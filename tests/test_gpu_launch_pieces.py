"""Calls launched in pieces, on the GPU: the same bits as in one launch, and rows past what one grid holds."""
import contextlib
import ctypes as C

import numpy as np
import pytest

import kv_plain as P

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _pieces(hip, n):
    """launches of at most n workgroups"""
    f = hip.lib().aoship_internal_set_launch_most
    f.restype, f.argtypes = C.c_uint32, [C.c_uint32]
    f(n)
    try:
        yield
    finally:
        f(0)


@pytest.mark.parametrize("most", [1, 7, 64])
@pytest.mark.parametrize("new", [[1] * 9, [40, 1, 0, 70, 1, 1, 1, 33, 2], [300, 1, 1, 1, 1, 1, 1, 1, 1]])
def test_weights(hip, most, new):
    import torch

    rng = np.random.default_rng(most)
    lens, nkv, nh, hd = [700, 1, 64, 900, 1500, 20, 4, 33, 2], 2, 6, 64
    pool = P.Pool(hip, lens, nkv, hd, 64, "mxfp8")
    k = P.to_gpu(P.bf16(rng.standard_normal((sum(lens), nkv, hd))))
    pool.cache.append(0, pool.batch(lens, lens), k, k)
    q = P.to_gpu(P.bf16(rng.standard_normal((sum(new), nh, hd))))
    got = [torch.full((9, nkv, 1500), 7.0, device="cuda") for _ in range(2)]
    pool.cache.weigh(0, pool.batch(new, lens), q, got[0])
    with _pieces(hip, most):
        pool.cache.weigh(0, pool.batch(new, lens), q, got[1])
    assert torch.equal(*got) and pool.cache.faults() == 0


@pytest.mark.parametrize("most", [1, 5])
@pytest.mark.parametrize("L", [300, 5000, 20000])
def test_evict(hip, most, L):
    import torch

    rng = np.random.default_rng(L)
    lens, keep, nkv, hd = [L, 200], [L // 3, 150], 3, 64
    pages = [-(-k // 64) for k in keep]
    pool = P.Pool(hip, lens, nkv, hd, 64, "mxfp4", spare=2 * sum(pages))
    k = P.to_gpu(P.bf16(rng.standard_normal((sum(lens), nkv, hd))))
    pool.cache.append(0, pool.batch(lens, lens), k, k)
    w = torch.rand((2, nkv, L), device="cuda")
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = []
    for i in range(2):
        to = np.full((2, max(pages)), -1, np.int32)
        for s, n in enumerate(pages):
            at = i * sum(pages) + s * pages[0]
            to[s, :n] = pool.spare[at:at + n]
        to = torch.from_numpy(to).cuda()
        kept, wo = dev(np.full((2, nkv, max(keep)), -7)), torch.full((2, nkv, L), 7.0, device="cuda")
        with _pieces(hip, most if i else 0):
            pool.cache.evict(0, pool.batch(lens, lens), w, dev(keep), to, kept, first=2, recent=9, weights_out=wo)
        back = [torch.empty((sum(keep), nkv, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        pool.cache.read(0, hip.KVBatch(dev([0, keep[0], sum(keep)]), dev(keep), to, max(keep), max(keep)), *back)
        got.append((kept, wo, *back))
    assert all(torch.equal(a, b) for a, b in zip(*got)) and pool.cache.faults() == 0


@pytest.mark.parametrize("most", [1, 3, 100])
@pytest.mark.parametrize("T,V", [(1, 50000), (3, 9001), (700, 40)])
def test_logprobs(hip, most, T, V):
    """Pieces that end within a row's slices too"""
    import torch

    x = torch.randn((T, V), device="cuda")
    t = torch.randint(0, V, (T,), device="cuda").int()
    op, got = hip.LogProbs(), []
    for n in (0, most, most):
        lp, ent = (torch.full((T,), 7.0, device="cuda") for _ in range(2))
        rank, ids = (torch.full(s, 7, dtype=torch.int32, device="cuda") for s in ((T,), (T, 5)))
        tops = torch.full((T, 5), 7.0, device="cuda")
        with _pieces(hip, n):
            op(x, t, lp, ent, rank, ids, tops)
        got.append((lp, ent, rank, ids, tops))
    assert all(torch.equal(a, b) for g in got[1:] for a, b in zip(got[0], g))


def test_logprobs_of_more_rows_than_a_grid_holds(hip):
    import torch

    T = (1 << 24) + 5  # times 256 threads: past 2^32
    x = torch.zeros((T, 2), device="cuda")
    x[:, 0] = torch.arange(T, device="cuda") % 64 / 16.0
    t = (torch.arange(T, device="cuda") % 2).int()
    lp, rank = torch.full((T,), 7.0, device="cuda"), torch.full((T,), 7, dtype=torch.int32, device="cuda")
    hip.LogProbs()(x, t, lp, rank=rank)
    z = x.double()
    want = torch.where(t == 0, z[:, 0], z[:, 1]) - torch.log(torch.exp(z[:, 0]) + torch.exp(z[:, 1]))
    # two exponentials and their sum, a logarithm and two subtractions, of magnitudes up to 4
    assert float((lp - want).abs().max()) <= 2.0 ** -24 * 30
    assert torch.equal(rank, t)  # (the first logit is the larger, or equal and first)
