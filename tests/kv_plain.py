"""Plain float64 forms of the paged key/value cache's operators, and the caches and batches that its tests use."""
import numpy as np

FORMATS = ("bf16", "mxfp8", "mxfp4")


def bf16(x):
    """float64 array -> the nearest bfloat16 values, ties to even (NaN and infinities as they are). A float32 step in
    between cannot round twice: callers pass float32 values or values exact in float32."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    nan = (u & 0x7FFFFFFF) > 0x7F800000
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32)
    r[nan] = 0x7FC00000
    return r.view(np.float32).astype(np.float64)


def quantised(x, fmt):
    """The values that a cache of format fmt holds of rows x [..., hd] of bfloat16 values."""
    if fmt == "bf16":
        return x.copy()
    top, low, mant, least = (448.0, -6, 3, -117) if fmt == "mxfp8" else (6.0, 0, 1, -125)
    out = np.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        blk = x[..., b:b + 32]
        with np.errstate(all="ignore"):
            amax = np.abs(blk).max(-1, keepdims=True)
            fin = np.isfinite(amax)  # (a NaN among them makes the maximum NaN)
            m = np.where(fin, amax, 1.0)
            frac, e = np.frexp(m / top)  # m / top = frac 2^e, frac in [0.5, 1)
            e = np.where(frac == 0.5, e - 1, e)  # the smallest e with m <= top 2^e
            e = np.maximum(np.where(m == 0, least, e), least)
            y = blk * 2.0 ** -e.astype(np.float64)
            p = np.frexp(np.where(np.isfinite(y), y, 0.0))[1] - 1
            grid = 2.0 ** (np.maximum(p, low) - mant).astype(np.float64)
            v = np.rint(y / grid) * grid * 2.0 ** e.astype(np.float64)
            v = np.where(np.abs(v) >= 2.0 ** 128, np.copysign(np.inf, v), v)  # (past the largest bfloat16)
        out[..., b:b + 32] = np.where(fin, v, np.nan)
    return out


def rotated(x, cos, sin):
    """float32 rows [T, heads, hd] -> rotated halves, each float32 operation rounded on its own"""
    h = x.shape[-1] // 2
    a, b = x[..., :h].astype(np.float32), x[..., h:].astype(np.float32)
    c, s = cos[:, None].astype(np.float32), sin[:, None].astype(np.float32)
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def attention(q, k, v, scale, window=0):
    """One sequence: q [n, nh, hd] are its last n positions, k and v [L, nkv, hd] float64 of all of them. Returns
    (o, a): the result and, for bounds, the same sum over |v|."""
    n, nh, hd = q.shape
    L, nkv = k.shape[0], k.shape[1]
    o, a = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    pos = np.arange(L - n, L)
    with np.errstate(all="ignore"):
        for t in range(n):
            if pos[t] < 0:
                continue
            lo = max(0, pos[t] + 1 - window) if window else 0
            for h in range(nh):
                kk, vv = k[lo:pos[t] + 1, h // (nh // nkv)], v[lo:pos[t] + 1, h // (nh // nkv)]
                s = kk @ q[t, h] * scale
                p = np.exp(s - s.max())
                p = p / p.sum()
                o[t, h], a[t, h] = p @ vv, p @ np.abs(vv)
    return o, a


def attention_bound(q, k, a, o, scale):
    """How far a result may be from attention(): it is rounded to bfloat16 (half a step: 2^-8 of it); each probability
    is rounded to bfloat16 before the second product (2^-8 of it, so 2^-8 of a); scores are float32 sums of exact
    products: hd additions and the scaling, each off by at most 2^-24 of sum |q| |k| scale =: S, which changes a
    probability by at most e^d - 1 <= 1.1 d, d = (hd + 4) 2^-24 S, and its normaliser as much again; exponentials and
    float32 sums of up to 2^17 terms in pieces: 2^-14 in all."""
    S = abs(scale) * np.abs(q).sum(-1).max(initial=0.0) * np.abs(np.where(np.isfinite(k), k, 0)).max(initial=0.0)
    d = (q.shape[-1] + 4) * 2.0 ** -24 * S
    return 2.0 ** -8 * np.abs(o) + (2.0 ** -8 + 2.2 * d + 2.0 ** -14) * a + 1e-30


class Pool:
    """A cache with its sequences' pages, dealt out in a shuffled order."""

    def __init__(self, hip, lens, nkv, hd, page, fmt, layers=1, spare=2, seed=0):
        import torch

        self.hip, self.page = hip, page
        count = [-(-n // page) for n in lens]
        order = np.random.default_rng(seed).permutation(sum(count) + spare)
        self.table = np.full((len(lens), max([1] + count) + 1), -1, np.int32)
        at = 0
        for s, n in enumerate(count):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        self.cache = hip.KVCache(layers, nkv, hd, page, sum(count) + spare, fmt)
        self.pages = torch.from_numpy(self.table).cuda()

    def batch(self, new, lens, max_new=None, max_len=None, starts=None):
        import torch

        st = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if starts is None else np.asarray(starts, np.int32)
        return self.hip.KVBatch(torch.from_numpy(st).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), self.pages,
                                max(new) if max_new is None else max_new, max(lens) if max_len is None else max_len)


def to_gpu(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda().bfloat16()


def to_cpu(t):
    return t.float().cpu().numpy().astype(np.float64)
