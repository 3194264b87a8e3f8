"""The measured operators of a paged key/value cache: writing new tokens into it and reading them
back (bfloat16, 8-bit or 4-bit), and attention of each sequence's new tokens over it.

  cache      one layer's new q, k and v rows (as the projections leave them) get their biases and
             their rotary embedding, k and v are quantised and written to the sequences' pages, and
             rows are read back as the values the cache stands for (KVCache.append, KVCache.read)
  attention  the new tokens' queries attend, causally and within an optional window, to everything
             the pages of their sequence hold (KVCache.attention): one token a sequence, a few
             drafted ones, a chunk of a prompt, a whole prompt, or a batch that mixes them

A row is quantised in blocks of 32 dimensions: a power-of-two scale, the smallest that keeps the
block's largest magnitude within the code's range, and e4m3 (8 bits, up to 448) or e2m1 (4 bits, up
to 6) codes, rounded to nearest even.
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
        # one user's next token: the smallest call, all launch and latency
        dict(name="cache 1 token", kind="cache", **H7B, page=64, format="bf16", seqs=1, new=1, past=511, ragged=0,
             ones=0, read="new", bias=True, packed=False),
        # a few users' prompts in one call, into a 4-bit cache, the projections' rows side by side
        dict(name="cache 5 prompts 4-bit", kind="cache", **H7B, page=128, format="mxfp4", seqs=5, new=1531, past=700,
             ragged=3, ones=0, read="new", bias=True, packed=True),
        # a long prompt of the largest model, 16-bit cache
        dict(name="cache prompt 8191", kind="cache", **H32B, page=256, format="bf16", seqs=1, new=8191, past=0,
             ragged=0, ones=0, read="new", bias=False, packed=True),
        # 16 streams write a token each and are then read back whole (to move them off the GPU)
        dict(name="cache read 16 streams", kind="cache", **H3B, page=64, format="mxfp8", seqs=16, new=1, past=8000,
             ragged=5, ones=0, read="all", bias=False, packed=False),
        # the most frequent attention call of all: one user's next token over a short context
        dict(name="attention 1 x 512", kind="attention", **H7B, page=64, format="bf16", seqs=1, new=1, past=511,
             ragged=0, ones=0, window=0),
        # a busy server's decode step: 32 streams of their own lengths, 8-bit cache
        dict(name="attention 32 streams 8-bit", kind="attention", **H3B, page=64, format="mxfp8", seqs=32, new=1,
             past=8190, ragged=7, ones=0, window=0),
        # the largest decode step: 64 long streams of a 16-bit cache
        dict(name="attention 64 streams", kind="attention", **H7B, page=128, format="bf16", seqs=64, new=1,
             past=16000, ragged=11, ones=0, window=0),
        # few streams of very long documents, 4-bit cache
        dict(name="attention 24 long 4-bit", kind="attention", **H32B, page=256, format="mxfp4", seqs=24, new=1,
             past=32767, ragged=13, ones=0, window=0),
        # drafted tokens to be verified, five a stream, small model
        dict(name="attention 12 x 5 drafted", kind="attention", **H05B, page=64, format="bf16", seqs=12, new=5,
             past=2000, ragged=0, ones=0, window=0),
        # a whole prompt
        dict(name="attention prompt 4076", kind="attention", **H7B, page=64, format="bf16", seqs=1, new=4076, past=0,
             ragged=0, ones=0, window=0),
        # the next chunk of a long prompt over what is cached of it, 8 bits
        dict(name="attention chunk 512 of 16384", kind="attention", **H32B, page=64, format="mxfp8", seqs=1, new=512,
             past=15872, ragged=0, ones=0, window=0),
        # a server's mixed step: chunks of four prompts among 28 decoding streams, windowed
        dict(name="attention mixed 32", kind="attention", **H3B, page=64, format="mxfp8", seqs=32, new=700,
             past=3500, ragged=17, ones=28, window=2048),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    c = dict(kind=rng.choice(["cache", "attention", "attention"]))
    c.update(rng.choice([H05B, H3B, H7B, H32B, dict(heads=8, kv_heads=8, head_dim=96),
                         dict(heads=16, kv_heads=2, head_dim=256), dict(heads=9, kv_heads=3, head_dim=80)]))
    c.update(page=rng.choice([64, 128, 256]), format=rng.choice(list(BITS)), ragged=rng.randrange(1, 10000))
    c["seqs"] = between(1, 64)
    style = rng.choice(["ones", "few", "chunk", "mixed"])
    c["new"] = {"ones": 1, "few": rng.randrange(2, 17), "chunk": between(17, 4000), "mixed": between(17, 1000)}[style]
    c["ones"] = c["seqs"] * 3 // 4 if style == "mixed" else 0
    if style == "chunk":
        c["seqs"] = between(1, 6)
    # at most as much cache as the largest listed case has, and half as much for chunks
    room = min(600000, 1200000000 // _row_bytes(c)) // c["seqs"] // (2 if c["new"] > 16 else 1)
    c["past"] = min(between(1, 32000), room) if rng.random() < 0.9 else 0
    while c["new"] > 16 and 4 * c["seqs"] * c["new"] * (c["past"] + c["new"]) * c["heads"] * c["head_dim"] > 1.6e11:
        c["new"], c["past"] = c["new"] * 3 // 4, c["past"] * 3 // 4
    if c["kind"] == "cache":
        c.update(read=rng.choice(["new", "all"]), bias=rng.random() < 0.5, packed=rng.random() < 0.5)
        if c["read"] == "all":
            c["past"] = min(c["past"], 120000 // c["seqs"])
    else:
        c.update(window=rng.choice([0, 0, between(100, 8000)]))
    return c


def _sizes(c):
    """(new tokens, positions held before them) of each sequence: the case's own, whatever the seed."""
    rng = random.Random("%s %d %d %d" % (c["ragged"], c["seqs"], c["new"], c["past"]))
    new, past = [], []
    for i in range(c["seqs"]):
        n = 1 if i < c["ones"] else c["new"]
        if c["ragged"] and i + 1 < c["seqs"]:  # (the last sequence is the longest)
            n = n if n <= 16 else rng.randint(n // 3, n)
            past.append(rng.randint(c["past"] // 4, c["past"]))
        else:
            past.append(c["past"])
        new.append(n)
    return new, past


def _seen(new, past, window):
    """(pairs of a new token and a position it sees, positions that some new token sees)"""
    pairs = reach = 0
    for n, p in zip(new, past):
        first = max(0, p + 1 - window) if window else 0
        reach += p + n - first
        short = max(0, min(n, window - p)) if window else n  # tokens that see everything before them
        pairs += sum(p + t + 1 for t in (0, short - 1)) * short // 2 if short else 0
        pairs += (n - short) * window
    return pairs, reach


def _row_bytes(c):
    """bytes of a position's keys and values in the cache"""
    scales = 0 if c["format"] == "bf16" else (c["head_dim"] + 31) // 32
    return 2 * c["kv_heads"] * (c["head_dim"] * BITS[c["format"]] // 8 + scales)


def work(c):
    new, past = _sizes(c)
    T, held = sum(new), sum(new) + sum(past)
    hd, nh, nkv = c["head_dim"], c["heads"], c["kv_heads"]
    row = _row_bytes(c)
    if c["kind"] == "cache":
        back = held if c["read"] == "all" else T
        return {"bytes": T * (2 * (2 * nh + 2 * nkv) * hd + row) + back * (row + 4 * nkv * hd),
                "flops": T * 8 * (nh + 2 * nkv) * hd}
    pairs, reach = _seen(new, past, c["window"])
    return {"bytes": 4 * T * nh * hd + reach * row, "flops": 4 * pairs * nh * hd}


def _rows(c, gen, n):
    """n new rows of k and of v: unit values, with some channels of the keys several times larger"""
    shape = (n, c["kv_heads"], c["head_dim"])
    k = torch.randn(shape, generator=gen, device=DEV)
    k[..., :: 13] *= 3.0
    return k.bfloat16(), torch.randn(shape, generator=gen, device=DEV).bfloat16()


def _inputs(c, seed):
    """What a call's inputs are made of, from the seed: the rows that the cache holds already (all
    sequences' in order), the new rows, biases, the rotary tables and which page is whose."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    new, past = _sizes(c)
    T, hd = sum(new), c["head_dim"]
    d = dict(new=new, past=past, T=T)
    d["old_k"], d["old_v"] = _rows(c, gen, sum(past))
    q = 1.5 * torch.randn((T, c["heads"], hd), generator=gen, device=DEV)
    k, v = _rows(c, gen, T)
    if c.get("packed"):
        both = torch.cat([q.bfloat16(), k, v], dim=1)
        nh, nkv = c["heads"], c["kv_heads"]
        d["q"], d["k"], d["v"] = both[:, :nh], both[:, nh:nh + nkv], both[:, nh + nkv:]
    else:
        d["q"], d["k"], d["v"] = q.bfloat16(), k, v
    d["qb"], d["kb"], d["vb"] = (
        0.5 * torch.randn((h, hd), generator=gen, device=DEV) if c.get("bias") else None
        for h in (c["heads"], c["kv_heads"], c["kv_heads"]))
    lens = [n + p for n, p in zip(new, past)]
    angle = torch.arange(max(lens), dtype=torch.float64, device=DEV)[:, None] * (
        THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd))
    d["cos"], d["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    count = [(n + c["page"] - 1) // c["page"] for n in lens]
    order = torch.randperm(sum(count) + 3, generator=gen, device=DEV).int()  # (pages of others too)
    pages = torch.full((len(lens), max(count)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, n in enumerate(count):
        pages[s, :n] = order[at:at + n]
        at += n
    d.update(lens=lens, pages=pages, num_pages=sum(count) + 3)
    return d


def _starts(counts):
    return torch.tensor([0] + list(counts), device=DEV).cumsum(0).int()


def prepare(c, seed):
    d = _inputs(c, seed)
    new, past, lens, hd, nkv = d["new"], d["past"], d["lens"], c["head_dim"], c["kv_heads"]
    st = dict(c=c, **{n: d[n] for n in ("q", "k", "v", "qb", "kb", "vb", "T", "pages")})
    st["starts"], st["lens"] = _starts(new), torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["max_new"], st["max_len"] = max(new), max(lens)
    whole = c["kind"] == "cache" and c["read"] == "all"
    st["back_starts"] = _starts(lens) if whole else st["starts"]
    back = sum(lens) if whole else d["T"]
    if own:
        sys.path.insert(0, str(ROOT / "adapter-os_amd"))
        import aoship

        aoship.init(0)
        cache = aoship.KVCache(1, nkv, hd, c["page"], d["num_pages"], c["format"])
        if sum(past):  # what earlier calls left in the cache
            held = aoship.KVBatch(_starts(past), torch.tensor(past, dtype=torch.int32, device=DEV), d["pages"],
                                  max(past), max(past))
            cache.append(0, held, d["old_k"], d["old_v"])
        if c["kind"] == "cache":
            cache.set_rope(d["cos"].cpu().numpy(), d["sin"].cpu().numpy())
            st["out"] = torch.zeros_like(d["q"], memory_format=torch.contiguous_format)
            st["k_back"] = torch.zeros((back, nkv, hd), dtype=torch.bfloat16, device=DEV)
            st["v_back"] = torch.zeros_like(st["k_back"])
        else:
            batch = aoship.KVBatch(st["starts"], st["lens"], d["pages"], st["max_new"], st["max_len"])
            cache.append(0, batch, d["k"], d["v"])
            st["out"] = torch.zeros((d["T"], c["heads"], hd), dtype=torch.bfloat16, device=DEV)
        st["batch"] = aoship.KVBatch(st["starts"], st["lens"], d["pages"], st["max_new"], st["max_len"])
        st["back"] = aoship.KVBatch(st["back_starts"], st["lens"], d["pages"], max(lens) if whole else max(new),
                                    st["max_len"])
        st["cache"] = cache
        aoship.sync()
        return st
    # the same cache as plain tensors of codes and scales, [page][position][head][...]
    st.update(cos=d["cos"], sin=d["sin"])
    wide = {"bf16": hd, "mxfp8": hd, "mxfp4": (hd + 1) // 2}[c["format"]]
    kind = torch.bfloat16 if c["format"] == "bf16" else torch.uint8
    for n in ("k", "v"):
        st[n + "_codes"] = torch.zeros((d["num_pages"] * c["page"], nkv, wide), dtype=kind, device=DEV)
        st[n + "_scales"] = torch.zeros((d["num_pages"] * c["page"], nkv, (hd + 31) // 32), dtype=torch.uint8, device=DEV)
    if sum(past):
        where = _slots(st, _starts(past), torch.tensor(past, device=DEV), sum(past))
        _store(st, "k", where, d["old_k"].float())
        _store(st, "v", where, d["old_v"].float())
    if c["kind"] == "attention":
        where = _slots(st, st["starts"], st["lens"], d["T"])
        _store(st, "k", where, d["k"].float())
        _store(st, "v", where, d["v"].float())
    return st


# ---- the plain form ---------------------------------------------------------------------------


def _tokens(starts, lens, T):
    """(sequence, position) of each of the T rows of a batch"""
    row = torch.arange(T, device=DEV)
    seq = (row[:, None] >= starts[None, 1:]).sum(1)
    return seq, (lens.long() - (starts[1:] - starts[:-1]).long())[seq] + row - starts.long()[seq]


def _slots(st, starts, lens, T):
    seq, pos = _tokens(starts, lens, T)
    page = st["c"]["page"]
    return st["pages"][seq, pos // page].long() * page + pos % page


def _blocks(x):
    """[..., hd] as [..., blocks, 32], the last block filled up with zeros"""
    pad = -x.shape[-1] % 32
    x = torch.cat([x, torch.zeros((*x.shape[:-1], pad), device=x.device)], dim=-1) if pad else x
    return x.view(*x.shape[:-1], -1, 32)


def _store(st, name, where, x):
    """Quantises float32 rows (of bfloat16 values) and writes their codes and scales."""
    fmt, hd = st["c"]["format"], st["c"]["head_dim"]
    if fmt == "bf16":
        st[name + "_codes"][where] = x.bfloat16()
        return
    b = _blocks(x)
    top = b.abs().amax(-1)
    frac, expo = torch.frexp(top)  # top = frac 2^expo, frac in [0.5, 1)
    if fmt == "mxfp8":
        e = (expo - 1 - 8 + (frac > 0.875).int()).clamp_min(-117)
    else:
        e = (expo - 1 - 2 + (frac > 0.75).int()).clamp_min(-125)
    e = torch.where(top == 0, torch.full_like(e, -117 if fmt == "mxfp8" else -125), e)
    t = torch.ldexp(b, -e[..., None]).reshape(*x.shape[:-1], -1)[..., :hd]
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


def _load(st, name, where):
    """The float32 values of the rows at `where` (any shape) of the cache."""
    fmt, hd = st["c"]["format"], st["c"]["head_dim"]
    codes = st[name + "_codes"][where]
    if fmt == "bf16":
        return codes.float()
    if fmt == "mxfp8":
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        value = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
        x = torch.stack([value[(codes & 15).long()], value[(codes >> 4).long()]], dim=-1).flatten(-2)
    scale = torch.ldexp(torch.ones((), device=DEV), st[name + "_scales"][where].int() - 127)
    return x * scale.repeat_interleave(32, dim=-1)[..., :hd]


def _rotate(st, x, pos):
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, a * s + b * c], dim=-1)


def _cache_plain(st):
    _, pos = _tokens(st["starts"], st["lens"], st["T"])
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if st["qb"] is not None:
        q, k, v = q + st["qb"], k + st["kb"], v + st["vb"]
    where = _slots(st, st["starts"], st["lens"], st["T"])
    _store(st, "k", where, _rotate(st, k, pos).bfloat16().float())
    _store(st, "v", where, v.bfloat16().float())
    back = int(st["lens"].sum()) if st["c"]["read"] == "all" else st["T"]
    where = _slots(st, st["back_starts"], st["lens"], back)
    return dict(q=_rotate(st, q, pos).bfloat16(), k=_load(st, "k", where).bfloat16(),
                v=_load(st, "v", where).bfloat16())


def _attention_plain(st):
    c = st["c"]
    nh, nkv, hd, g = c["heads"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    n, most, lmax = st["lens"].numel(), st["max_new"], st["max_len"]
    j = torch.arange(lmax, device=DEV)
    where = st["pages"][:, j // c["page"]].long().clamp_min(0) * c["page"] + j % c["page"]  # [n, lmax]
    held = (j < st["lens"][:, None])[:, :, None, None]
    k = torch.where(held, _load(st, "k", where), 0.0).permute(0, 2, 3, 1).contiguous()  # [n, nkv, hd, lmax]
    v = torch.where(held, _load(st, "v", where), 0.0).permute(0, 2, 1, 3).contiguous()
    t = torch.arange(most, device=DEV)
    count = st["starts"][1:] - st["starts"][:-1]
    row = (st["starts"][:-1, None] + t).clamp_max(st["T"] - 1).long()  # [n, most]
    q = st["q"].float()[row].view(n, most, nkv, g, hd).permute(0, 2, 1, 3, 4).reshape(n, nkv, most * g, hd)
    at = (st["lens"] - count)[:, None] + t  # the tokens' positions
    sees = j <= at[:, :, None]
    if c["window"]:
        sees = sees & (j > at[:, :, None] - c["window"])
    sees = sees[:, None, :, None, :]  # [n, 1, most, 1, lmax]
    s = (torch.matmul(q, k) * (hd ** -0.5)).view(n, nkv, most, g, lmax)
    s = torch.where(sees, s, float("-inf"))
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3.0e38))
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n, nkv, most * g, lmax), v).view(n, nkv, most, g, hd) / total.clamp_min(1e-30)
    o = o.permute(0, 2, 1, 3, 4).reshape(n, most, nh, hd)
    return o[t < count[:, None]].bfloat16()


def run(st):
    c = st["c"]
    if c["kind"] == "cache":
        if not own:
            return _cache_plain(st)
        st["cache"].append(0, st["batch"], st["k"], st["v"], q=st["q"], q_out=st["out"], k_bias=st["kb"],
                           v_bias=st["vb"], q_bias=st["qb"])
        st["cache"].read(0, st["back"], st["k_back"], st["v_back"])
        return dict(q=st["out"], k=st["k_back"], v=st["v_back"])
    if not own:
        return dict(out=_attention_plain(st))
    st["cache"].attention(0, st["batch"], st["q"], st["out"], window=c["window"])
    return dict(out=st["out"])


# ---- the definition in 64 bits ----------------------------------------------------------------


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
    hd, nkv, g = c["head_dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    half, fmt = hd // 2, c["format"]
    if c["kind"] == "cache":
        pos = torch.cat([torch.arange(p, p + n, device=DEV) for n, p in zip(d["new"], d["past"])])
        turn = torch.complex(d["cos"].double()[pos], d["sin"].double()[pos])[:, None]

        def full(x, bias, rotated):
            x = x.double() + (0.0 if bias is None else bias.double())
            if not rotated:
                return x
            z = torch.complex(x[..., :half], x[..., half:]) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        k, v = _quantised(full(d["k"], d["kb"], True), fmt), _quantised(full(d["v"], d["vb"], False), fmt)
        if c["read"] == "all":
            old_k, old_v = _quantised(d["old_k"].double(), fmt), _quantised(d["old_v"].double(), fmt)
            k, v = (torch.cat([piece for o, n in zip(old.split(d["past"]), fresh.split(d["new"])) for piece in (o, n)])
                    for old, fresh in ((old_k, k), (old_v, v)))
        return dict(q=full(d["q"], d["qb"], True), k=k, v=v)
    outs, t0, p0 = [], 0, 0
    for n, p in zip(d["new"], d["past"]):
        k = _quantised(torch.cat([d["old_k"][p0:p0 + p], d["k"][t0:t0 + n]]).double(), fmt)
        v = _quantised(torch.cat([d["old_v"][p0:p0 + p], d["v"][t0:t0 + n]]).double(), fmt)
        q = d["q"][t0:t0 + n].double()
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)[None]
        hidden = (far < 0) | ((far >= c["window"]) if c["window"] else False)
        o = torch.empty((n, c["heads"], hd), dtype=torch.float64, device=DEV)
        for h in range(c["heads"]):
            s = (q[:, h] @ k[:, h // g].T) / math.sqrt(hd)
            o[:, h] = torch.softmax(s.masked_fill(hidden, float("-inf")), dim=-1) @ v[:, h // g]
        outs.append(o)
        t0, p0 = t0 + n, p0 + p
    return dict(out=torch.cat(outs))
