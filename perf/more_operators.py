"""The measured operators around the attention over a paged key/value cache, as a serving step uses them:

  rotary    new q, k and v rows whose rotary positions the caller gives, on up to three axes (time, height and width
            of images and video), rotated and written to the sequences' pages; read back as the values the cache
            holds (KVCache.append with positions, KVCache.read)
  weights   the attention weight that each cached position gets from the batch's rows, summed over the rows and over
            the query heads that share a key/value head (KVCache.weigh)
  evict     of each sequence and key/value head the first positions, the last ones and those of greatest weight
            between are kept, moved in order to other pages, and read back (KVCache.evict, KVCache.read)
  logprobs  of rows of logits: the log probability and the rank of a given token, the entropy, and the most probable
            tokens (LogProbs)

A cache holds rows in bfloat16, or in blocks of 32 dimensions: a power-of-two scale, the smallest that keeps the
block's largest magnitude within the code's range, and e4m3 (8 bits, up to 448) or e2m1 (4 bits, up to 6) codes.
"""
import math
import random
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent

own = False

DEV = "cuda:0"
THETA = 1.0e6
BITS = {"bf16": 16, "mxfp8": 8, "mxfp4": 4}
H05B = dict(heads=14, kv_heads=2, head_dim=64)
H3B = dict(heads=24, kv_heads=8, head_dim=128)
H7B = dict(heads=28, kv_heads=4, head_dim=128)
H32B = dict(heads=40, kv_heads=8, head_dim=128)
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a decode step of 48 streams whose prompts held images: one token each, positions of their own
        dict(name="rotary 48 streams", kind="rotary", **H7B, page=64, format="bf16", seqs=48, new=1, past=1500, ragged=1,
             bias=True, weave=False, wide=20),
        # two prompts with video, into an 8-bit cache
        dict(name="rotary video 2 x 6111", kind="rotary", **H3B, page=128, format="mxfp8", seqs=2, new=6111, past=0,
             ragged=2, bias=False, weave=True, wide=34),
        # one user's next token over a short context: the smallest call, all launch and latency
        dict(name="weights 1 x 512", kind="weights", **H7B, page=64, format="bf16", seqs=1, new=1, past=511, ragged=0,
             window=0, prior=True),
        # a step of 64 long streams, the weights of earlier steps added to
        dict(name="weights 64 streams", kind="weights", **H7B, page=128, format="bf16", seqs=64, new=1, past=16000,
             ragged=3, window=0, prior=True),
        # the last 32 tokens of twelve prompts say what of them to keep, 8-bit cache
        dict(name="weights 12 x 32 observed", kind="weights", **H3B, page=64, format="mxfp8", seqs=12, new=32, past=8100,
             ragged=4, window=0, prior=False),
        # all tokens of a prompt
        dict(name="weights prompt 4001", kind="weights", **H7B, page=64, format="bf16", seqs=1, new=4001, past=0,
             ragged=0, window=0, prior=False),
        # a small model's stream comes down to half
        dict(name="evict 1 x 2047", kind="evict", **H05B, page=64, format="bf16", seqs=1, past=2047, ragged=0, keep=1000,
             first=4, recent=128),
        # sixteen streams down to 4096 positions each, 4-bit cache
        dict(name="evict 16 x 12000 4-bit", kind="evict", **H3B, page=64, format="mxfp4", seqs=16, past=12000, ragged=5,
             keep=4096, first=4, recent=512),
        # four long documents of the largest model to less than half, 16-bit cache
        dict(name="evict 4 x 32767", kind="evict", **H32B, page=256, format="bf16", seqs=4, past=32767, ragged=6,
             keep=15000, first=0, recent=2000),
        # one sampled token with five alternatives: the smallest call
        dict(name="logprobs 1 row", kind="logprobs", rows=1, vocab=152064, format="f32", top=5, spare=0),
        # a step of 64 streams with twenty alternatives each
        dict(name="logprobs 64 rows", kind="logprobs", rows=64, vocab=128256, format="f32", top=20, spare=0),
        # prompts to be scored, bfloat16 logits of an odd vocabulary (many ties)
        dict(name="logprobs 4000 rows bf16", kind="logprobs", rows=4000, vocab=50257, format="bf16", top=10, spare=3),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotary", "weights", "weights", "evict", "logprobs"])
    if kind == "logprobs":
        c = dict(kind=kind, vocab=between(300, 160000), format=rng.choice(["f32", "bf16"]), top=rng.choice([0, 1, 5, 20, 32]),
                 spare=rng.choice([0, 0, 1, 64]))
        c["rows"] = between(1, max(1, min(6000, 100000000 // c["vocab"])))
        return c
    c = dict(kind=kind)
    c.update(rng.choice([H05B, H3B, H7B, H32B, dict(heads=8, kv_heads=8, head_dim=96),
                         dict(heads=16, kv_heads=2, head_dim=256), dict(heads=9, kv_heads=3, head_dim=80)]))
    c.update(page=rng.choice([64, 128, 256]), format=rng.choice(list(BITS)), ragged=rng.randrange(1, 10000))
    row = _row_bytes(c)
    if kind == "rotary":
        c["seqs"] = between(1, 64)
        c["new"] = 1 if rng.random() < 0.3 else between(2, max(2, min(6000, 9500 // c["seqs"])))
        c["past"] = between(1, max(1, 60000 // c["seqs"])) if rng.random() < 0.8 else 0
        c.update(bias=rng.random() < 0.5, weave=rng.random() < 0.5, wide=rng.randrange(3, 60))
        return c
    if kind == "evict":
        c["seqs"] = between(1, 32)
        c["past"] = between(100, min(40000, 120000 // c["seqs"], 400000000 // row // c["seqs"]))
        c["keep"] = max(3, int(c["past"] * rng.uniform(0.05, 1.05)))
        c["first"] = rng.choice([0, 1, 4])
        c["recent"] = rng.randrange(0, c["keep"] - c["first"])
        return c
    c["seqs"] = between(1, 64)
    style = rng.choice(["ones", "few", "prompt"])
    c["new"] = {"ones": 1, "few": rng.randrange(2, 65), "prompt": between(65, 4000)}[style]
    if style != "ones":
        c["seqs"] = between(1, 12 if style == "few" else 4)
    room = min(600000, 1200000000 // row) // c["seqs"] // (1 if style == "ones" else 4)
    c["past"] = min(between(1, 32000), room) if rng.random() < 0.9 else 0
    while c["new"] > 1 and 2 * c["seqs"] * c["new"] * (c["past"] + c["new"]) * c["heads"] * c["head_dim"] > 6.0e10:
        c["new"], c["past"] = (c["new"] + 1) // 2, c["past"] * 3 // 4
    c.update(window=rng.choice([0, 0, between(100, 8000)]), prior=rng.random() < 0.5)
    return c


def _sizes(c):
    """(new tokens, positions held before them) of each sequence: the case's own, whatever the seed."""
    rng = random.Random("%s %d %d %d" % (c["ragged"], c["seqs"], c.get("new", 0), c["past"]))
    new, past = [], []
    for i in range(c["seqs"]):
        n = c.get("new", 0)
        if c["ragged"] and i + 1 < c["seqs"]:  # (the last sequence is the longest)
            new.append(n if n <= 64 else rng.randint(n // 3, n))
            past.append(rng.randint(c["past"] // 4, c["past"]))
        else:
            new.append(n)
            past.append(c["past"])
    return new, past


def _row_bytes(c):
    """bytes of a position's keys and values in the cache"""
    scales = 0 if c["format"] == "bf16" else (c["head_dim"] + 31) // 32
    return 2 * c["kv_heads"] * (c["head_dim"] * BITS[c["format"]] // 8 + scales)


def work(c):
    if c["kind"] == "logprobs":
        size = c["rows"] * c["vocab"]
        return {"bytes": size * (4 if c["format"] == "f32" else 2) + c["rows"] * (16 + 8 * c["top"]), "flops": 8 * size}
    new, past = _sizes(c)
    T, row, hd, nh, nkv = sum(new), _row_bytes(c), c["head_dim"], c["heads"], c["kv_heads"]
    if c["kind"] == "rotary":
        return {"bytes": T * (2 * (2 * nh + 2 * nkv) * hd + 2 * row + 4 * nkv * hd + 12), "flops": T * 8 * (nh + 2 * nkv) * hd}
    if c["kind"] == "evict":
        held, kept = sum(past), sum(min(c["keep"], p) for p in past)
        # weights in and out, the rows kept read, written and read back
        return {"bytes": nkv * (8 * held + 4 * kept) + kept * (3 * row + 4 * nkv * hd), "flops": held * nkv}
    pairs = reach = 0
    for n, p in zip(new, past):
        first = max(0, p + 1 - c["window"]) if c["window"] else 0
        reach += p + n - first
        for t in (range(n) if c["window"] else ()):
            pairs += min(p + t + 1, c["window"])
        pairs += 0 if c["window"] else n * p + n * (n + 1) // 2
    held = T + sum(past)
    return {"bytes": 2 * T * nh * hd + reach * row // 2 + held * nkv * (8 if c["prior"] else 4), "flops": 2 * pairs * nh * hd}


def _starts(counts):
    return torch.tensor([0] + list(counts), device=DEV).cumsum(0).int()


def _rows(c, gen, n):
    """n rows of k and of v: unit values, with some channels of the keys several times larger"""
    shape = (n, c["kv_heads"], c["head_dim"])
    k = torch.randn(shape, generator=gen, device=DEV)
    k[..., :: 13] *= 3.0
    return k.bfloat16(), torch.randn(shape, generator=gen, device=DEV).bfloat16()


def _axes(c):
    """the axis (0 time, 1 height, 2 width) of each rotated pair: runs of pairs, or in turn"""
    half = c["head_dim"] // 2
    return [i % 3 if c["weave"] else (0 if 4 * i < half else 1 if 8 * i < 5 * half else 2) for i in range(half)]


def _positions(c, new, past):
    """[3, tokens]: text (all axes alike), then frames of `wide` columns and half as many rows, then text"""
    out = []
    for n, p in zip(new, past):
        i = torch.arange(n, device=DEV)
        if n < 10:
            out.append((p + i).expand(3, n))
            continue
        lead, tail, w = n // 10, n // 10, c["wide"]
        h = (w + 1) // 2
        j = (i - lead).clamp(0, n - lead - tail - 1)
        grid = p + lead + torch.stack([j // (w * h), j // w % h, j % w])
        text = p + lead + max((n - lead - tail - 1) // (w * h) + 1, h, w) + (i - (n - tail))
        out.append(torch.where(i < lead, p + i, torch.where(i < n - tail, grid, text)))
    return torch.cat(out, dim=1).int()


def _pages(c, lens, gen, first=0):
    """([sequences, pages] of shuffled numbers from `first` on, -1 past each sequence's own; the numbers taken)"""
    count = [(n + c["page"] - 1) // c["page"] for n in lens]
    order = (torch.randperm(sum(count) + 3, generator=gen, device=DEV) + first).int()  # (pages of others too)
    pages = torch.full((len(lens), max(count)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(count):
        pages[s, :n] = order[at:at + n]
        at += n
    return pages, sum(count) + 3


def _inputs(c, seed):
    """What a call's inputs are made of, from the seed."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "logprobs":
        T, V = c["rows"], c["vocab"]
        x = 2.5 * torch.randn((T, V + c["spare"]), generator=gen, device=DEV)
        ids = torch.randint(0, V, (T, 4), generator=gen, device=DEV)
        x.scatter_add_(1, ids, 6.0 + 4.0 * torch.rand((T, 4), generator=gen, device=DEV))  # (likely tokens)
        x[:, V - V // 100:V] = float("-inf")  # numbers that stand for no token
        other = torch.randint(0, V - V // 100, (T,), generator=gen, device=DEV)
        targets = torch.where(torch.rand(T, generator=gen, device=DEV) < 0.6, ids[:, 0], other).int()
        x = x if c["format"] == "f32" else x.bfloat16()
        return dict(logits=x[:, :V], targets=targets)
    new, past = _sizes(c)
    T, hd = sum(new), c["head_dim"]
    lens = [n + p for n, p in zip(new, past)]
    d = dict(new=new, past=past, T=T, lens=lens)
    d["old_k"], d["old_v"] = _rows(c, gen, sum(past))
    d["pages"], d["num_pages"] = _pages(c, lens, gen)
    if c["kind"] == "evict":
        d["kept"] = [min(c["keep"], n) for n in lens]
        d["to"], more = _pages(c, d["kept"], gen, d["num_pages"])
        d["num_pages"] += more
        shape = (len(lens), c["kv_heads"], max(lens))
        w = torch.rand(shape, generator=gen, device=DEV) ** 9 * 30.0
        w = torch.where(torch.rand(shape, generator=gen, device=DEV) < 0.2, 0.0, w)  # (never looked at: ties)
        d["weights"] = torch.where(torch.arange(max(lens), device=DEV) < torch.tensor(lens, device=DEV)[:, None, None], w, 0.0)
        return d
    d["q"] = (1.5 * torch.randn((T, c["heads"], hd), generator=gen, device=DEV)).bfloat16()
    d["k"], d["v"] = _rows(c, gen, T)
    if c["kind"] == "weights":
        if c["prior"]:
            w = 5.0 * torch.rand((len(lens), c["kv_heads"], max(lens)), generator=gen, device=DEV)
            w = torch.where(torch.arange(max(lens), device=DEV) < torch.tensor(past, device=DEV)[:, None, None], w, 0.0)
            d["prior"] = w
        return d
    d["qb"], d["kb"], d["vb"] = (
        0.5 * torch.randn((h, hd), generator=gen, device=DEV) if c["bias"] else None
        for h in (c["heads"], c["kv_heads"], c["kv_heads"]))
    d["at"] = _positions(c, new, past)
    angle = torch.arange(int(d["at"].max()) + 1, dtype=torch.float64, device=DEV)[:, None] * (
        THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd))
    d["cos"], d["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    return d


def prepare(c, seed):
    d = _inputs(c, seed)
    if c["kind"] == "logprobs":
        st = dict(c=c, **d)
        if own:
            sys.path.insert(0, str(ROOT / "adapter-os_amd"))
            import aoship

            aoship.init(0)
            T, n = c["rows"], c["top"]
            st["op"] = aoship.LogProbs()
            st["logprob"], st["entropy"] = (torch.zeros(T, device=DEV) for _ in range(2))
            st["rank"] = torch.zeros(T, dtype=torch.int32, device=DEV)
            st["ids"] = torch.zeros((T, n), dtype=torch.int32, device=DEV) if n else None
            st["tops"] = torch.zeros((T, n), device=DEV) if n else None
        return st
    new, past, lens, hd, nkv = d["new"], d["past"], d["lens"], c["head_dim"], c["kv_heads"]
    st = dict(c=c, **d)
    st["starts"], st["lens_dev"] = _starts(new), torch.tensor(lens, dtype=torch.int32, device=DEV)
    if c["kind"] == "evict":
        st["keep"] = torch.full((len(lens),), c["keep"], dtype=torch.int32, device=DEV)
        st["kept_starts"], st["kept_lens"] = _starts(d["kept"]), torch.tensor(d["kept"], dtype=torch.int32, device=DEV)
        st["kept_pos"] = torch.full((len(lens), nkv, max(d["kept"])), -1, dtype=torch.int32, device=DEV)
    if own:
        sys.path.insert(0, str(ROOT / "adapter-os_amd"))
        import aoship

        aoship.init(0)
        cache = aoship.KVCache(1, nkv, hd, c["page"], d["num_pages"], c["format"])
        if sum(past):  # what earlier calls left in the cache
            held = aoship.KVBatch(_starts(past), torch.tensor(past, dtype=torch.int32, device=DEV), d["pages"],
                                  max(past), max(past))
            cache.append(0, held, d["old_k"], d["old_v"])
        st["batch"] = aoship.KVBatch(st["starts"], st["lens_dev"], d["pages"], max(new), max(lens))
        back = d["T"]
        if c["kind"] == "rotary":
            cache.set_rope(d["cos"].cpu().numpy(), d["sin"].cpu().numpy())
            cache.set_rope_axes(_axes(c))
            st["out"] = torch.zeros_like(d["q"])
            st["back"] = st["batch"]
        elif c["kind"] == "weights":
            cache.append(0, st["batch"], d["k"], d["v"])
            cache.reserve_weigh(c["heads"], st["batch"], d["T"])
            st["weights"] = torch.zeros((len(lens), nkv, max(lens)), device=DEV)
        else:
            st["weights_out"] = torch.zeros_like(d["weights"])
            st["back"] = aoship.KVBatch(st["kept_starts"], st["kept_lens"], d["to"], max(d["kept"]), max(d["kept"]))
            back = sum(d["kept"])
        if c["kind"] != "weights":
            st["k_back"] = torch.zeros((back, nkv, hd), dtype=torch.bfloat16, device=DEV)
            st["v_back"] = torch.zeros_like(st["k_back"])
        st["cache"] = cache
        aoship.sync()
        return st
    # the same cache as plain tensors of codes and scales, [page][position][head][...]
    wide = {"bf16": hd, "mxfp8": hd, "mxfp4": (hd + 1) // 2}[c["format"]]
    kind = torch.bfloat16 if c["format"] == "bf16" else torch.uint8
    for n in ("k", "v"):
        st[n + "_codes"] = torch.zeros((d["num_pages"] * c["page"], nkv, wide), dtype=kind, device=DEV)
        st[n + "_scales"] = torch.zeros((d["num_pages"] * c["page"], nkv, (hd + 31) // 32), dtype=torch.uint8, device=DEV)
    if sum(past):
        where = _slots(st, d["pages"], _starts(past), torch.tensor(past, device=DEV), sum(past))
        _store(st, "k", where, d["old_k"].float())
        _store(st, "v", where, d["old_v"].float())
    if c["kind"] == "weights":
        _store(st, "k", _slots(st, d["pages"], st["starts"], st["lens_dev"], d["T"]), d["k"].float())
    return st


# ---- the plain forms --------------------------------------------------------------------------


def _slots(st, pages, starts, lens, T):
    """where in the cache each of the T rows of a batch is"""
    row = torch.arange(T, device=DEV)
    seq = (row[:, None] >= starts[None, 1:]).sum(1)
    pos = (lens.long() - (starts[1:] - starts[:-1]).long())[seq] + row - starts.long()[seq]
    return pages[seq, pos // st["c"]["page"]].long() * st["c"]["page"] + pos % st["c"]["page"]


def _store(st, name, where, x):
    """Quantises float32 rows (of bfloat16 values) and writes their codes and scales."""
    fmt, hd = st["c"]["format"], st["c"]["head_dim"]
    if fmt == "bf16":
        st[name + "_codes"][where] = x.bfloat16()
        return
    pad = -hd % 32
    b = torch.cat([x, torch.zeros((*x.shape[:-1], pad), device=DEV)], dim=-1).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    frac, expo = torch.frexp(top)  # top = frac 2^expo, frac in [0.5, 1)
    most, low, full = (8, -117, 0.875) if fmt == "mxfp8" else (2, -125, 0.75)
    e = (expo - 1 - most + (frac > full).int()).clamp_min(low)
    e = torch.where(top == 0, torch.full_like(e, low), e)
    t = torch.ldexp(b, -e[..., None]).flatten(-2)[..., :hd]
    if fmt == "mxfp8":
        codes = t.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        mag = t.abs()
        step = torch.where(mag < 2.0, 0.5, torch.where(mag < 4.0, 1.0, 2.0))
        halves = (torch.round(mag / step) * step * 2.0).long()  # 0 1 2 3 4 6 8 12
        code = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8, device=DEV)[halves]
        code = code | ((t.view(torch.int32) < 0).to(torch.uint8) << 3)
        codes = code[..., 0::2] | (code[..., 1::2] << 4)
    st[name + "_codes"][where] = codes
    st[name + "_scales"][where] = (e + 127).to(torch.uint8)


def _values(c, codes, scales):
    """The float32 values that codes and scales stand for."""
    if c["format"] == "bf16":
        return codes.float()
    if c["format"] == "mxfp8":
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        value = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
        x = torch.stack([value[(codes & 15).long()], value[(codes >> 4).long()]], dim=-1).flatten(-2)
    scale = torch.ldexp(torch.ones((), device=DEV), scales.int() - 127)
    return x * scale.repeat_interleave(32, dim=-1)[..., :c["head_dim"]]


def _load(st, name, where):
    return _values(st["c"], st[name + "_codes"][where], st[name + "_scales"][where])


def _rotary_plain(st):
    c = st["c"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if st["qb"] is not None:
        q, k, v = q + st["qb"], k + st["kb"], v + st["vb"]
    row = st["at"].long()[torch.tensor(_axes(c), device=DEV)].T  # [tokens, pairs]: the table row of each pair
    pair = torch.arange(c["head_dim"] // 2, device=DEV)
    cos, sin = st["cos"][row, pair][:, None], st["sin"][row, pair][:, None]

    def turned(x):
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1).bfloat16()

    where = _slots(st, st["pages"], st["starts"], st["lens_dev"], st["T"])
    _store(st, "k", where, turned(k).float())
    _store(st, "v", where, v.bfloat16().float())
    return dict(q=turned(q), k=_load(st, "k", where).bfloat16(), v=_load(st, "v", where).bfloat16())


def _weights_plain(st):
    c = st["c"]
    nkv, hd, g, lmax = c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], max(st["lens"])
    out = torch.zeros((len(st["lens"]), nkv, lmax), device=DEV)
    j = torch.arange(lmax, device=DEV)
    if c["new"] == 1:  # one row a sequence: all of them together
        where = st["pages"][:, j // c["page"]].long().clamp_min(0) * c["page"] + j % c["page"]  # [n, lmax]
        k = _load(st, "k", where).permute(0, 2, 3, 1).contiguous()  # [n, nkv, hd, lmax]
        s = torch.matmul(st["q"].float().unflatten(1, (nkv, g)), k) * (hd ** -0.5)  # [n, nkv, g, lmax]
        sees = j < st["lens_dev"][:, None]
        if c["window"]:
            sees = sees & (j >= st["lens_dev"][:, None] - c["window"])
        s = torch.where(sees[:, None, None], s, float("-inf"))
        s = torch.exp(s - s.amax(-1, keepdim=True))
        out = (s / s.sum(-1, keepdim=True)).sum(2)
    else:
        at = 0
        for i, (n, p) in enumerate(zip(st["new"], st["past"])):
            L = n + p
            where = st["pages"][i, j[:L] // c["page"]].long() * c["page"] + j[:L] % c["page"]
            k = _load(st, "k", where).permute(1, 2, 0).contiguous()  # [nkv, hd, L]
            q = st["q"][at:at + n].float().unflatten(1, (nkv, g)).permute(1, 0, 2, 3)  # [nkv, n, g, hd]
            far = (p + torch.arange(n, device=DEV))[:, None] - j[:L]
            hidden = (far < 0) | ((far >= c["window"]) if c["window"] else False)
            for h in range(nkv):
                s = torch.matmul(q[h].reshape(n * g, hd), k[h]).view(n, g, L) * (hd ** -0.5)
                s = s.masked_fill(hidden[:, None], float("-inf"))
                s = torch.exp(s - s.amax(-1, keepdim=True))
                out[i, h, :L] = (s / s.sum(-1, keepdim=True)).sum((0, 1))
            at += n
    return dict(weights=out + st["prior"] if c["prior"] else out)


def _evict_plain(st):
    c = st["c"]
    L = st["lens_dev"][:, None, None]
    j = torch.arange(max(st["lens"]), device=DEV)
    count = torch.minimum(st["keep"], st["lens_dev"])[:, None, None]
    must = (j < c["first"]) | (j >= L - c["recent"])
    rank = torch.where(must, float("inf"), st["weights"])
    rank = torch.where(j < L, rank, float("-inf"))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :max(st["kept"])]
    i = torch.arange(order.shape[-1], device=DEV)
    pos = torch.sort(torch.where(i < count, order, 1 << 30), dim=-1).values  # [n, nkv, most], in order
    live = i < count
    pos = torch.where(live, pos, 0)
    w = torch.zeros_like(st["weights"])
    w[..., :pos.shape[-1]] = torch.where(live, torch.gather(st["weights"], -1, pos), 0.0)
    # each kept row to its new place: source and destination slots [n, nkv, most]
    seq = torch.arange(len(st["lens"]), device=DEV)[:, None, None]
    src = st["pages"][seq, pos // c["page"]].long() * c["page"] + pos % c["page"]
    dst = st["to"][seq, i // c["page"]].long() * c["page"] + i % c["page"]
    live, dst = live.expand_as(pos), dst.expand_as(pos)
    head = torch.arange(c["kv_heads"], device=DEV)[:, None].expand_as(pos)
    for n in ("k_codes", "k_scales", "v_codes", "v_scales"):
        st[n][dst[live], head[live]] = st[n][src[live], head[live]]
    back = _slots(st, st["to"], st["kept_starts"], st["kept_lens"], sum(st["kept"]))
    return dict(kept=torch.where(live, pos, -1).int(), weights=w, k=_load(st, "k", back).bfloat16(),
                v=_load(st, "v", back).bfloat16())


def _logprobs_plain(st):
    c = st["c"]
    x, t = st["logits"].float(), st["targets"].long()[:, None]
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    entropy = (torch.log(total) - (e * d.clamp_min(-1000.0)).sum(1, keepdim=True) / total)[:, 0]
    base = top + torch.log(total)
    mine = torch.gather(x, 1, t)
    i = torch.arange(c["vocab"], device=DEV)
    rank = ((x > mine) | ((x == mine) & (i < t))).sum(1).int()
    out = dict(logprob=(mine - base)[:, 0], entropy=entropy, rank=rank)
    if c["top"]:
        ids, vals, left = [], [], x.clone()
        for _ in range(c["top"]):
            best = left.amax(1, keepdim=True)
            at = torch.where(left == best, i, c["vocab"]).amin(1, keepdim=True)
            left.scatter_(1, at, float("-inf"))
            ids.append(at)
            vals.append(best - base)
        out.update(ids=torch.cat(ids, 1).int(), tops=torch.cat(vals, 1))
    return out


def run(st):
    c = st["c"]
    if not own:
        return {"rotary": _rotary_plain, "weights": _weights_plain, "evict": _evict_plain,
                "logprobs": _logprobs_plain}[c["kind"]](st)
    if c["kind"] == "logprobs":
        st["op"](st["logits"], st["targets"], logprob=st["logprob"], entropy=st["entropy"], rank=st["rank"],
                 top_ids=st["ids"], top_logprobs=st["tops"])
        out = dict(logprob=st["logprob"], entropy=st["entropy"], rank=st["rank"])
        if c["top"]:
            out.update(ids=st["ids"], tops=st["tops"])
        return out
    if c["kind"] == "weights":
        st["cache"].weigh(0, st["batch"], st["q"], st["weights"], window=c["window"], prior=st.get("prior"))
        return dict(weights=st["weights"])
    if c["kind"] == "evict":
        st["cache"].evict(0, st["batch"], st["weights"], st["keep"], st["to"], st["kept_pos"], first=c["first"],
                          recent=c["recent"], weights_out=st["weights_out"])
        st["cache"].read(0, st["back"], st["k_back"], st["v_back"])
        return dict(kept=st["kept_pos"], weights=st["weights_out"], k=st["k_back"], v=st["v_back"])
    st["cache"].append(0, st["batch"], st["k"], st["v"], q=st["q"], q_out=st["out"], k_bias=st["kb"], v_bias=st["vb"],
                       q_bias=st["qb"], positions=st["at"])
    st["cache"].read(0, st["back"], st["k_back"], st["v_back"])
    return dict(q=st["out"], k=st["k_back"], v=st["v_back"])


# ---- the definitions in 64 bits ---------------------------------------------------------------


def _quantised(x, fmt):
    """float64 rows as the values that a cache of this format holds of them"""
    x = x.bfloat16().double()
    if fmt == "bf16":
        return x
    top_code, low, mantissa, least = (448.0, -6, 3, -117) if fmt == "mxfp8" else (6.0, 0, 1, -125)
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        blk = x[..., b:b + 32]
        top = blk.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / top_code))
        e = torch.where(top > top_code * torch.exp2(e), e + 1, e)
        e = torch.where(top <= top_code * torch.exp2(e - 1), e - 1, e).clamp_min(least)
        e = torch.where(top == 0, torch.full_like(e, least), e)
        y = blk / torch.exp2(e)
        power = torch.floor(torch.log2(y.abs().clamp_min(1e-300))).clamp_min(low)
        power = torch.where(torch.exp2(power + 1) <= y.abs(), power + 1, power)
        grid = torch.exp2(power - mantissa)
        out[..., b:b + 32] = torch.round(y / grid) * grid * torch.exp2(e)
    return out


def exact(c, seed):
    d = _inputs(c, seed)
    if c["kind"] == "logprobs":
        parts = []
        for x, t in zip(d["logits"].split(500), d["targets"].long().split(500)):
            lp = torch.log_softmax(x.double(), dim=1)
            p = torch.exp(lp)
            mine = lp.gather(1, t[:, None])
            raw = x.gather(1, t[:, None])
            before = torch.arange(c["vocab"], device=DEV)[None] < t[:, None]
            rank = (x > raw).sum(1) + ((x == raw) & before).sum(1)
            r = dict(logprob=mine[:, 0], entropy=-torch.where(p > 0, p * lp, 0.0).sum(1), rank=rank.int())
            if c["top"]:
                ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]]
                r.update(ids=ids.int(), tops=lp.gather(1, ids))
            parts.append(r)
        return {n: torch.cat([r[n] for r in parts]) for n in parts[0]}
    hd, nkv, g, fmt = c["head_dim"], c["kv_heads"], c["heads"] // c["kv_heads"], c["format"]
    if c["kind"] == "rotary":
        pairs = torch.arange(hd // 2, device=DEV)
        at = torch.stack([d["at"][a].long() for a in _axes(c)], dim=1)
        turn = torch.complex(d["cos"].double()[at, pairs], d["sin"].double()[at, pairs])[:, None]

        def full(x, bias, rotated):
            x = x.double() + (0.0 if bias is None else bias.double())
            if not rotated:
                return x
            z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        return dict(q=full(d["q"], d["qb"], True), k=_quantised(full(d["k"], d["kb"], True), fmt),
                    v=_quantised(full(d["v"], d["vb"], False), fmt))
    if c["kind"] == "evict":
        n, most = len(d["lens"]), max(d["kept"])
        kept = torch.full((n, nkv, most), -1, dtype=torch.int32, device=DEV)
        weights = torch.zeros((n, nkv, max(d["lens"])), dtype=torch.float64, device=DEV)
        ks, vs, at = [], [], 0
        for s, (L, m) in enumerate(zip(d["lens"], d["kept"])):
            k, v = (_quantised(d[x][at:at + L].double(), fmt) for x in ("old_k", "old_v"))
            at += L
            rows = torch.empty((2, m, nkv, hd), dtype=torch.float64, device=DEV)
            for h in range(nkv):
                w = d["weights"][s, h, :L].double()
                free = torch.arange(min(c["first"], L), max(L - c["recent"], min(c["first"], L)), device=DEV)
                best = free[torch.sort(-w[free], stable=True).indices[:max(0, m - (L - free.numel()))]]
                outer = torch.ones(L, dtype=torch.bool, device=DEV)
                outer[free] = False
                pos = torch.cat([torch.nonzero(outer)[:, 0], best]).sort().values
                kept[s, h, :m], weights[s, h, :m] = pos.int(), w[pos]
                rows[0, :, h], rows[1, :, h] = k[pos, h], v[pos, h]
            ks.append(rows[0])
            vs.append(rows[1])
        return dict(kept=kept, weights=weights, k=torch.cat(ks), v=torch.cat(vs))
    out = torch.zeros((len(d["lens"]), nkv, max(d["lens"])), dtype=torch.float64, device=DEV)
    t0 = p0 = 0
    for s, (n, p) in enumerate(zip(d["new"], d["past"])):
        k = _quantised(torch.cat([d["old_k"][p0:p0 + p], d["k"][t0:t0 + n]]).double(), fmt)
        q = d["q"][t0:t0 + n].double()
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)[None]
        hidden = (far < 0) | ((far >= c["window"]) if c["window"] else False)
        for h in range(c["heads"]):
            x = (q[:, h] @ k[:, h // g].T) / math.sqrt(hd)
            out[s, h // g, :p + n] += torch.softmax(x.masked_fill(hidden, float("-inf")), dim=-1).sum(0)
        t0, p0 = t0 + n, p0 + p
    return dict(weights=out + d["prior"].double() if c["prior"] else out)
