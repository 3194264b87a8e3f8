"""Model.score on the GPU, row by row against float64 of the same logits.

The models' layers add nothing to the residual stream (their last projections are zero), embeddings are -1 and 1 and the
final norm's weights are powers of two, so that the LM head's input is known exactly: its logits are then exact sums in
float64, and what the kernels make of them is off by their float32 sums alone."""
import numpy as np
import pytest

import oracle

pytestmark = pytest.mark.gpu

V = 2592  # 81 row blocks of the LM head: not a multiple of what a workgroup takes


def _model(hip, H, seed, max_seq=256):
    """(model, exact logits of every token [V, V] float64, how far a logit may be off [V, V])"""
    rng = np.random.default_rng(seed)
    nh, hd, inter = 2, 32, 128
    m = hip.Model(1, H, inter, nh, 1, hd, V, max_seq, 10000.0, 1e-6)
    emb = np.where(rng.random((V, H)) < 0.5, -1.0, 1.0).astype(np.float32)
    m.set_embedding(rows_bf16=(emb.view(np.uint32) >> 16).astype(np.uint16))

    def q4(out, inp):
        packed = rng.integers(0, 2 ** 32, (out, inp // 8), dtype=np.uint32)
        s = rng.uniform(0.01, 0.02, (out, inp // 64)).astype(np.float16)
        return packed, s, (-8.0 * s.astype(np.float32)).astype(np.float16)

    def zeros(out, inp):
        return np.zeros((out, inp // 8), np.uint32), np.zeros((out, inp // 64), np.float16), np.zeros((out, inp // 64), np.float16)

    for name, out, inp in (("q_proj", nh * hd, H), ("k_proj", hd, H), ("v_proj", hd, H), ("gate_proj", inter, H),
                           ("up_proj", inter, H)):
        m.layers[0].set_base(name, *q4(out, inp))
    m.layers[0].set_base("o_proj", *zeros(H, nh * hd))
    m.layers[0].set_base("down_proj", *zeros(H, inter))
    for which in (0, 1):
        m.set_norm(0, which, np.ones(H, np.float32))
    norm = 2.0 ** rng.integers(-1, 2, H)
    m.set_norm(-1, 0, norm.astype(np.float32))
    packed, s, b = q4(V, H)
    m.set_lm_head(packed, s, b)
    m.set_adapters([])
    # a row's root mean square is (1 + 1e-6)^(1/2), which bfloat16 does not see
    x = emb.astype(np.float64) * norm
    codes = ((packed[:, :, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(V, H).astype(np.float64)
    s, b = s.astype(np.float64), b.astype(np.float64)
    logits, size = np.zeros((V, V)), np.zeros((V, V))
    for g in range(H // 64):
        c, xg = codes[:, 64 * g:64 * g + 64], x[:, 64 * g:64 * g + 64]
        t, sx = xg @ c.T, xg.sum(1)[:, None]  # exact
        logits += t * s[:, g] + sx * b[:, g]
        # the kernels multiply codes offset by 128 (sums exact in float32) and take the offset off with the bias
        size += np.abs(t + 128 * sx) * s[:, g] + np.abs(sx * (b[:, g] - 128 * s[:, g]))
    # two fused operations a group, and the joins of its waves' and workgroups' sums (32 at most), each half a step
    return m, logits, 2.0 ** -24 * (2 * (H // 64) + 32) * size


def _score(hip, m, ids, targets, n):
    import torch

    T = len(ids)
    dev = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
    lp, ent = torch.full((T,), 7.0, device="cuda"), torch.full((T,), 7.0, device="cuda")
    rank, top = torch.full((T,), -7, dtype=torch.int32, device="cuda"), torch.full((T, n), -7, dtype=torch.int32, device="cuda")
    tops, last = torch.full((T, n), 7.0, device="cuda"), torch.full((V,), 7.0, device="cuda")
    rings = torch.from_numpy(np.zeros(T, oracle.RING_DTYPE).view(np.uint8).copy()).cuda()
    m.score(dev(ids), rings, dev(targets), lp, ent, rank, top, tops, logits=last)
    torch.cuda.synchronize()
    return [x.cpu().numpy().astype(np.float64) for x in (lp, ent, rank, top, tops, last)]


def _lse(x):
    m = x.max(-1, keepdims=True)
    return m + np.log(np.exp(x - m).sum(-1, keepdims=True))


def _off(got, logits, tol, targets, n):
    """Rows whose answers are not those of these logits, each up to tol off (a distribution's logarithms then move by up to
    twice that, its entropy by 2 (1 + H) times that), beside what float32 does to the log probabilities (test_gpu_logprobs)."""
    lp, ent, rank, top, tops, _ = got
    T = len(lp)
    d = tol.max(1)
    f32 = 2.0 ** -24 * (V / 256 + 90 + 4 * 12)
    z = logits - _lse(logits)
    H = -(np.exp(z) * z).sum(1)
    own = logits[np.arange(T), targets]
    off = np.abs(lp - z[np.arange(T), targets]) > 2 * d + f32
    off |= np.abs(ent - H) > 2 * (1 + H) * (d + f32)
    off |= rank < (logits > own[:, None] + 2 * d[:, None]).sum(1)
    off |= rank > (logits >= own[:, None] - 2 * d[:, None]).sum(1) - 1
    order = -np.sort(-logits, axis=1)[:, :n]
    ok = (top >= 0) & (top < V)
    at = np.take_along_axis(logits, np.where(ok, top, 0).astype(int), 1)
    off |= (~ok | (np.abs(at - order) > 2 * d[:, None])).any(1)
    off |= (np.abs(tops - np.take_along_axis(z, np.where(ok, top, 0).astype(int), 1)) > (2 * d + f32)[:, None]).any(1)
    off |= np.array([len(set(r)) < n for r in top.tolist()])
    return off


@pytest.mark.parametrize("H", [128, 512, 1024, 2048])
def test_every_row_of_a_prompt(hip, H):
    """The LM head's kernels of one and two rows, of few, of 3 to 32 (from hidden 512 on those whose waves read their input
    themselves, whole and split) and of several passes of 32; every row, and no other row's answers."""
    m, logits, tol = _model(hip, H, H)
    rng = np.random.default_rng(1)
    n = 8
    for T in (1, 2, 3, 9, 17, 32, 33, 70, 130):
        print(f"hidden {H}, {T} rows", flush=True)
        m.reset_cache()
        ids, targets = rng.permutation(V)[:T], rng.integers(0, V, T)
        targets[::3] = logits[ids].argmax(1)[::3]
        got = _score(hip, m, ids, targets, n)
        off = _off(got, logits[ids], tol[ids], targets, n)
        assert not off.any(), np.flatnonzero(off)
        if T > 1:  # (that the bounds tell rows apart)
            turned = np.roll(ids, 1)
            assert _off(got, logits[turned], tol[turned], targets, n).all()
        assert (np.abs(got[5] - logits[ids[-1]]) <= tol[ids[-1]]).all()


def test_one_token_is_forwards_logits(hip):
    """Rows one at a time: the log probabilities of forward()'s own logits, ids and ranks exactly"""
    import torch

    from test_gpu_logprobs import _close, _plain

    m, _, _ = _model(hip, 512, 5)
    rng = np.random.default_rng(2)
    ids, targets = rng.permutation(V)[:6], rng.integers(0, V, 6)
    rings = torch.from_numpy(np.zeros(1, oracle.RING_DTYPE).view(np.uint8).copy()).cuda()
    last = torch.zeros(V, device="cuda")
    for i in range(6):
        got = _score(hip, m, ids[i:i + 1], targets[i:i + 1], 8)
        m.reset_cache()
        m.forward(torch.from_numpy(ids[i:i + 1].astype(np.int32)).cuda(), rings, last)
        m.reset_cache()
        x = last.double().cpu().numpy()
        assert np.array_equal(x, got[5])
        lp, rank, ent, top, tops = _plain(x[None], targets[i:i + 1], 8)
        _close(got[0], lp, V)
        _close(got[4], tops, V)
        assert abs(got[1][0] - ent[0]) <= 2.0 ** -24 * (V / 256 + 90) * (2 + 2 * ent[0])
        assert np.array_equal(got[2], rank) and np.array_equal(got[3], top)
