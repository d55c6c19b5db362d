"""The 4-bit weight and 8-bit cache operators of a decode step, as cases that can be timed and checked.

`run` is one pass: in plain elementary torch operations where `own` is false, through the public entry points of
`demonic_amd` where it is true.  Both read the same bytes: MXFP4 codes (two to a byte, low half first) with an E8M0
byte for each block of 32, and cache pages of e4m3 codes with an E8M0 byte for each page and head.

kind      entry points                          a pass is
quant     mxfp4_quantize, mxfp4_dequantize      rows to MXFP4 and the values the codes stand for, in bf16
product   gemv_mxfp4_rd                         y = x @ W', f32 x, W in MXFP4
product4  gemm_mxfp4                            y = x @ W', both in MXFP4
append    kv8_append                            new tokens' k and v into the pages of their sequences
attend    kv8_attend                            causal attention of each sequence's last tokens over its pages

Shapes are Llama-3-8B's, the repository's edge shapes (rows of 4097) and generic ones.
"""
import math
import random

import torch

own = False

HIDDEN, FFN, VOCAB = 4096, 14336, 128256    # Llama-3-8B
HEADS, KV_HEADS, DIM = 32, 8, 128
MAX_WEIGHT = VOCAB * HIDDEN                 # elements of the LM head
MAX_MACS = FFN * HIDDEN * 2048              # multiply-adds of the largest listed product
MAX_TOKENS = 64 * 8192                      # cached tokens, times KV_HEADS * DIM, of the largest listed decode
MAX_SCORES = 4 * 2048 * 8192 * HEADS * DIM  # multiply-adds of the listed prompt's scores
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a bf16 checkpoint's gate/up weight on its way to 4 bits
        {"name": "quant_weight", "kind": "quant", "rows": FFN, "k": HIDDEN, "dtype": "bf16"},
        # activations of a small batch at an odd row length: a few microseconds, so launches count
        {"name": "quant_odd", "kind": "quant", "rows": 33, "k": 4097, "dtype": "f32"},
        # one token against one GPU's share of gate/up under 8-way tensor parallelism: the smallest weight read alone
        {"name": "share_m1", "kind": "product", "m": 1, "n": 1792, "k": HIDDEN},
        # the LM head for a batch of 16 sequences: the largest weight
        {"name": "lm_head_m16", "kind": "product", "m": 16, "n": VOCAB, "k": HIDDEN},
        # a prompt of 512 tokens with f32 activations against gate/up
        {"name": "up_m512", "kind": "product", "m": 512, "n": FFN, "k": HIDDEN},
        # activations in 4 bits too: rows of odd length and an odd batch
        {"name": "w4a4_odd_m33", "kind": "product4", "m": 33, "n": 11008, "k": 4097},
        # a prompt of 2048 tokens against down, activations in 4 bits too
        {"name": "w4a4_m2048", "kind": "product4", "m": 2048, "n": HIDDEN, "k": FFN},
        # a decode step of 64 sequences puts one token each into its last page
        {"name": "append_decode", "kind": "append", "batch": 64, "new": 1, "len": 4096, "heads": KV_HEADS, "dim": DIM,
         "page": 64, "dtype": "f32"},
        # four prompts of up to 2048 tokens
        {"name": "append_prompt", "kind": "append", "batch": 4, "new": 2048, "len": 4096, "heads": KV_HEADS, "dim": DIM,
         "page": 64, "dtype": "bf16"},
        # one token of one long sequence: few rows, a long axis
        {"name": "attend_long", "kind": "attend", "batch": 1, "new": 1, "len": 131072, "q_heads": HEADS,
         "heads": KV_HEADS, "dim": DIM, "page": 64, "window": 0, "dtype": "f32"},
        # one token each of 64 sequences of uneven length
        {"name": "attend_batch", "kind": "attend", "batch": 64, "new": 1, "len": 8192, "q_heads": HEADS,
         "heads": KV_HEADS, "dim": DIM, "page": 64, "window": 0, "dtype": "bf16"},
        # prompt chunks of up to 2048 tokens of four sequences
        {"name": "attend_prompt", "kind": "attend", "batch": 4, "new": 2048, "len": 8192, "q_heads": HEADS,
         "heads": KV_HEADS, "dim": DIM, "page": 64, "window": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of [lo, hi], spread over its logarithm: mostly multiples of 128, some of 32, some odd."""
    v, u = _log(rng, lo, hi), rng.random()
    return max(lo, v // 128 * 128) if u < 0.6 else max(lo, v // 32 * 32) if u < 0.75 else v


def draw(rng):
    u = rng.random()
    while True:
        if u < 0.15:
            c = {"kind": "quant", "rows": _log(rng, 1, 16384), "k": _size(rng, 64, 16384),
                 "dtype": rng.choice(("f32", "bf16"))}
            if c["rows"] * c["k"] <= FFN * HIDDEN:
                return c
        elif u < 0.55:
            c = {"kind": "product" if u < 0.4 else "product4",
                 "m": _log(rng, 1, 16) if rng.random() < 0.5 else _log(rng, 17, 2048),
                 "n": _size(rng, 512, 131072), "k": _size(rng, 512, 16384)}
            w = c["n"] * c["k"]
            if w <= MAX_WEIGHT and w * c["m"] <= (MAX_MACS if u >= 0.4 else MAX_MACS // 4):
                return c
        else:
            group = rng.choice((1, 2, 4, 4, 7, 8))
            heads = rng.choice((1, 2, 4, 8, 8, 16))
            dim = rng.choice((64, 96, 128, 128, 128, 256))
            decode = rng.random() < 0.6
            c = {"kind": "append" if u < 0.7 else "attend", "batch": _log(rng, 1, 128 if decode else 8),
                 "new": 1 if decode else _log(rng, 2, 2048), "len": _log(rng, 64, 131072 if decode else 16384)}
            c["len"] = max(c["len"], c["new"])
            if c["kind"] == "attend":
                c.update(q_heads=group * heads, window=rng.choice((0, 0, 0, _log(rng, 16, 4096))))
            c.update(heads=heads, dim=dim, page=rng.choice((16, 32, 64, 64, 128)), dtype=rng.choice(("f32", "bf16")))
            kv, scores = c["batch"] * c["len"] * heads * dim, c["batch"] * c["new"] * c["len"] * heads * group * dim
            if kv <= MAX_TOKENS * KV_HEADS * DIM and scores <= MAX_SCORES // (4 if c["dtype"] == "f32" else 1):
                return c


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 29)
    return gen


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _packed(gen, rows, k, scale):
    """Rows of N(0, scale) in MXFP4, as the quantiser lays them out, in pieces that need little room."""
    q = torch.empty((rows, -(-k // 128) * 64), device="cuda", dtype=torch.uint8)
    s = torch.empty((rows, -(-k // 128) * 4), device="cuda", dtype=torch.uint8)
    step = max(1, (1 << 26) // k)
    for r in range(0, rows, step):
        x = _randn(gen, min(step, rows - r), k) * scale
        q[r:r + step], s[r:r + step] = _to_mxfp4(x)
    return q, s


def _spans(case):
    """Uneven sequences, the same for every seed: (lengths with the new tokens, new tokens).  The first is as long as
    the case says, the others have a quarter of that to all of it, and half to all of the new tokens."""
    new, most, rng = case["new"], case["len"], random.Random(5)
    news = [new] + [max(1, round(new * rng.uniform(0.5, 1))) for _ in range(case["batch"] - 1)]
    lens = [most] + [max(n, round(most * rng.uniform(0.25, 1))) for n in news[1:]]
    return lens, news


def _cache(case, seed):
    """The pages of a batch, filled: k with a few large channels, as keys have after their rotation."""
    gen = _gen(seed)
    lens, news = (torch.tensor(v, device="cuda", dtype=torch.int32) for v in _spans(case))
    starts = torch.cat([torch.zeros(1, device="cuda").int(), news.cumsum(0).int()])
    h, d, page = case["heads"], case["dim"], case["page"]
    width = -(-case["len"] // page)
    used = (lens + page - 1) // page
    pages = int(used.sum()) + 2
    ids = torch.randperm(pages, generator=gen, device="cuda").int()
    first = torch.cat([torch.zeros(1, device="cuda").int(), used.cumsum(0).int()[:-1]])
    at = torch.arange(width, device="cuda")[None]
    table = torch.where(at < used[:, None], ids[(first[:, None] + at).clamp(max=pages - 1).long()], -1).int()
    channel = torch.where(torch.rand(d, generator=gen, device="cuda") < 0.05, 6.0, 1.0)
    k = torch.empty((pages, h, page, d), device="cuda", dtype=torch.float8_e4m3fn)
    v = torch.empty((pages, h, d, page), device="cuda", dtype=torch.float8_e4m3fn)
    ks, vs = (torch.empty((pages, h), device="cuda", dtype=torch.uint8) for _ in range(2))
    step = max(1, (1 << 26) // (h * page * d))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        for x, codes, scales in ((_randn(gen, n, h, page, d) * channel, k, ks), (_randn(gen, n, h, d, page), v, vs)):
            e = _scale8(x.abs().amax((2, 3)))
            codes[p:p + step], scales[p:p + step] = _to_e4m3(x, e[..., None, None]), e
    return {"k": k, "v": v, "ks": ks, "vs": vs, "table": table, "lens": lens, "starts": starts}, gen, channel


def prepare(case, seed):
    kind = case["kind"]
    st = {"case": case}
    if kind == "quant":
        x = _randn(_gen(seed), case["rows"], case["k"]) * 0.02
        st["x"] = x.to(_dtype(case))
        rows, k = case["rows"], -(-case["k"] // 128)
        st["q"] = torch.empty((rows, k * 64), device="cuda", dtype=torch.uint8)
        st["s"] = torch.empty((rows, k * 4), device="cuda", dtype=torch.uint8)
        st["y"] = torch.empty((rows, case["k"]), device="cuda", dtype=torch.bfloat16)
    elif kind in ("product", "product4"):
        gen = _gen(seed)
        m, n, k = case["m"], case["n"], case["k"]
        st["wq"], st["ws"] = _packed(gen, n, k, 0.02)
        if kind == "product":
            st["x"] = _randn(gen, m, k)
        else:
            st["xq"], st["xs"] = _packed(gen, m, k, 1.0)
        st["y"] = torch.empty((m, n), device="cuda", dtype=torch.float32)
    else:
        cache, gen, channel = _cache(case, seed)
        st.update(cache)
        total = int(st["starts"][-1])
        if kind == "append":
            st["nk"] = (_randn(gen, total, case["heads"], case["dim"]) * channel).to(_dtype(case))
            st["nv"] = _randn(gen, total, case["heads"], case["dim"]).to(_dtype(case))
        else:
            st["q"] = _randn(gen, total, case["q_heads"], case["dim"]).to(_dtype(case))
            st["out"] = torch.empty_like(st["q"])
    torch.cuda.synchronize()  # the library runs on its own stream: its inputs are ready before the first call
    return st


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _two(e):
    """2^e in f32 for whole e of [-127, 127], from its bits (a power function need not be exact)."""
    e = e.int()
    return torch.where(e == -127, 1 << 22, (e + 127) << 23).view(torch.float32)


def _to_mxfp4(x):
    """(codes, scales) of f32 rows."""
    rows, k = x.shape
    wide = torch.zeros((rows, -(-k // 128) * 128), device=x.device, dtype=torch.float32)
    wide[:, :k] = x
    wide = wide.view(rows, -1, 32)
    amax = wide.abs().amax(2)
    e = ((amax.view(torch.int32) >> 23) - 129).clamp(-127, 127)  # floor(log2) - 2; subnormal amax: the least
    a = (wide * _two(-e)[..., None]).abs()
    code = (a > 0.25).byte()  # to nearest, ties to the even code
    for above, edge in ((False, 0.75), (True, 1.25), (False, 1.75), (True, 2.5), (False, 3.5), (True, 5.0)):
        code += (a > edge) if above else (a >= edge)
    code |= torch.signbit(wide).byte() << 3
    bad = ~torch.isfinite(amax)
    code = torch.where(bad[..., None], 0, code).view(rows, -1, 2)
    return code[..., 0] | code[..., 1] << 4, torch.where(bad, 255, e + 127).byte()


def _from_mxfp4(q, s, k):
    """f32 values [rows, k]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
    codes = torch.stack([q & 15, q >> 4], -1).view(q.shape[0], -1, 32)
    scale = torch.where(s == 255, math.nan, _two(s.int().clamp(max=254) - 127))
    return (table[codes.int()] * scale[..., None]).view(q.shape[0], -1)[:, :k]


def _scale8(amax):
    """The E8M0 byte of the least power of two 2^e with amax <= 448 * 2^e."""
    return (((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(0, 254).byte()


def _to_e4m3(x, scale):
    return (x * _two(127 - scale.int())).to(torch.float8_e4m3fn)


def _from_e4m3(codes, scale):
    return codes.float() * _two(scale.int() - 127)


def _append(st):
    """All pages that get tokens, at once: a page's earlier codes are rounded again where its scale grows."""
    c = st["case"]
    page, h, d = c["page"], c["heads"], c["dim"]
    lens, starts, table = st["lens"].long(), st["starts"].long(), st["table"]
    news = starts[1:] - starts[:-1]
    from_page = (lens - news) // page
    most = -(-c["new"] // page) + 1
    slots = from_page[:, None] + torch.arange(most, device=lens.device)[None]     # [b, most] pages of a sequence
    b, j = (slots * page < lens[:, None]).nonzero(as_tuple=True)
    slot = slots[b, j]
    ids = table[b, slot].long()
    pos = slot[:, None] * page + torch.arange(page, device=lens.device)[None]     # [n, page] positions
    first = (lens - news)[b][:, None]
    fresh, kept = (pos >= first) & (pos < lens[b][:, None]), pos < first
    row = (starts[b][:, None] + pos - first).clamp(0, st["nk"].shape[0] - 1)
    for name, new, flip in (("k", st["nk"], False), ("v", st["nv"], True)):
        codes, scales = st[name], st[name + "s"]
        x = torch.where(fresh[:, None, :, None], new[row].float().transpose(1, 2), 0.0)       # [n, h, page, d]
        old = codes[ids].transpose(2, 3) if flip else codes[ids]
        had = scales[ids]
        need = _scale8(x.abs().amax((2, 3)))
        e = torch.where(kept[:, :1], torch.maximum(had, need), need)
        before = _from_e4m3(old, had[..., None, None])
        out = torch.where(kept[:, None, :, None] & (e > had)[..., None, None],
                          _to_e4m3(before, e[..., None, None]).view(torch.uint8), old.view(torch.uint8))
        out = torch.where(fresh[:, None, :, None], _to_e4m3(x, e[..., None, None]).view(torch.uint8), out)
        codes.view(torch.uint8)[ids] = out.transpose(2, 3) if flip else out
        scales[ids] = e
    return {"k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}


def _attend(st):
    c = st["case"]
    b, h, d, page, n = c["batch"], c["heads"], c["dim"], c["page"], c["new"]
    group = c["q_heads"] // h
    lens, starts = st["lens"].long(), st["starts"].long()
    news = starts[1:] - starts[:-1]
    ids = st["table"].clamp(min=0).long()
    k = _from_e4m3(st["k"][ids], st["ks"][ids][..., None, None])                                # [b, w, h, page, d]
    k = k.permute(0, 2, 1, 3, 4).reshape(b * h, -1, d)
    v = _from_e4m3(st["v"][ids], st["vs"][ids][..., None, None])                                # [b, w, h, d, page]
    v = v.permute(0, 2, 1, 4, 3).reshape(b * h, -1, d)
    i = torch.arange(n, device=lens.device)
    row = (starts[:-1, None] + i[None]).clamp(max=st["q"].shape[0] - 1)                         # [b, n]
    q = st["q"].float()[row].view(b, n, h, group, d).permute(0, 2, 1, 3, 4).reshape(b * h, n * group, d)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * d ** -0.5
    at = (lens - news)[:, None] + i[None]                                                       # positions [b, n]
    j = torch.arange(k.shape[1], device=lens.device)
    sees = (j <= at[..., None]) & (st["table"] >= 0).repeat_interleave(page, 1)[:, None]
    if c["window"]:
        sees &= j > at[..., None] - c["window"]
    s = s.view(b, h, n, group, -1)
    s.masked_fill_(~sees[:, None, :, None], -math.inf)
    s = s - s.amax(-1, keepdim=True)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b * h, n * group, -1), v).view(b, h, n, group, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, h * group, d)
    return o[i[None] < news[:, None]].to(st["q"].dtype)


def run(st):
    c = st["case"]
    kind = c["kind"]
    if own:
        return _run_own(st)
    if kind == "quant":
        q, s = _to_mxfp4(st["x"].float())
        return {"values": _from_mxfp4(q, s, c["k"]).to(torch.bfloat16), "scales": s}
    if kind == "append":
        return _append(st)
    if kind == "attend":
        return _attend(st)
    x = st["x"] if kind == "product" else _from_mxfp4(st["xq"], st["xs"], c["k"])
    return torch.matmul(x, _from_mxfp4(st["wq"], st["ws"], c["k"]).t())


def _run_own(st):
    import demonic_amd as hip
    c = st["case"]
    kind = c["kind"]
    p = {n: t.data_ptr() for n, t in st.items() if isinstance(t, torch.Tensor)}
    if kind == "quant":
        hip.mxfp4_quantize(p["x"], p["q"], p["s"], c["rows"], c["k"], dtype=c["dtype"])
        hip.mxfp4_dequantize(p["q"], p["s"], p["y"], c["rows"], c["k"], dtype="bf16")
        return {"values": st["y"], "scales": st["s"]}
    if kind == "product":
        hip.gemv_mxfp4_rd(p["x"], p["wq"], p["ws"], p["y"], c["m"], c["k"], c["n"])
        return st["y"]
    if kind == "product4":
        hip.gemm_mxfp4(p["xq"], p["xs"], p["wq"], p["ws"], p["y"], c["m"], c["k"], c["n"])
        return st["y"]
    cache = hip.KV8Cache(p["k"], p["v"], p["ks"], p["vs"], st["k"].shape[0], c["heads"], c["page"], c["dim"])
    batch = hip.KV8Batch(p["table"], st["table"].shape[1], p["lens"], p["starts"], c["batch"], c["new"], c["len"])
    if kind == "append":
        hip.kv8_append(cache, batch, p["nk"], p["nv"], dtype=c["dtype"])
        return {"k": st["k"], "v": st["v"], "ks": st["ks"], "vs": st["vs"]}
    hip.kv8_attend(cache, batch, p["q"], p["out"], c["q_heads"], dtype=c["dtype"], window=c["window"])
    return st["out"]


# ---- work -----------------------------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quant":
        n, size = case["rows"] * case["k"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * (size + 2 * 17 / 32 + 2), "flops": 2 * n}
    if kind in ("product", "product4"):
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k * 17 / 32 + m * k * (4 if kind == "product" else 17 / 32) + 4 * m * n,
                "flops": 2 * m * n * k}
    size = 4 if case["dtype"] == "f32" else 2
    lens, news = _spans(case)
    row = case["heads"] * case["dim"]
    if kind == "append":
        return {"bytes": sum(news) * row * 2 * (size + 1), "flops": 4 * sum(news) * row}
    window = case["window"] or max(lens)
    seen = [min(l, window - 1 + n) for l, n in zip(lens, news)]
    pairs = sum(min(l - i, window) for l, n in zip(lens, news) for i in range(n))
    q = case["q_heads"] * case["dim"]
    return {"bytes": sum(seen) * row * 2 + 2 * sum(news) * q * size, "flops": 4 * pairs * q}


# ---- 64 bits --------------------------------------------------------------------------------------------------------

def _two64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values4(q, s, k):
    """f64 values of MXFP4 rows, from the format's definition: sign, two exponent bits, one of fraction."""
    c = torch.empty((q.shape[0], q.shape[1] * 2), device=q.device, dtype=torch.float64)
    for half in (0, 1):
        bits = (q >> (4 * half)).long() & 15
        ex, fr = (bits >> 1) & 3, (bits & 1).double()
        mag = torch.where(ex == 0, 0.5 * fr, (1 + 0.5 * fr) * _two64(ex - 1))
        c[:, half::2] = torch.where(bits >= 8, -mag, mag)
    return (c * _two64(s.long() - 127).repeat_interleave(32, 1))[:, :k]


def _nearest(x, bits, least):
    """f64 values to the nearest with `bits` bits of fraction and exponents from `least`, ties to even."""
    ex = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least)))
    step = _two64(ex.clamp(min=least) - bits)
    return torch.round(x / step) * step


def _least8(amax):
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448))
    e = torch.where(448 * _two64(e) < amax, e + 1, torch.where(448 * _two64(e - 1) >= amax, e - 1, e))
    return e.clamp(-127, 127)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        rows, k = case["rows"], case["k"]
        x = torch.zeros((rows, -(-k // 32) * 32), device="cuda", dtype=torch.float64)
        x[:, :k] = st["x"].double()
        x = x.view(rows, -1, 32)
        e = (torch.floor(torch.log2(x.abs().amax(2).clamp(min=1e-300))) - 2).clamp(-127, 127)
        unit = _two64(e)[..., None]
        return {"values": (_nearest(x / unit, 1, 0).clamp(-6, 6) * unit).view(rows, -1)[:, :k], "scales": None}
    if kind in ("product", "product4"):
        x = st["x"].double() if kind == "product" else _values4(st["xq"], st["xs"], case["k"])
        step = max(1, (1 << 26) // case["k"])
        return torch.cat([x @ _values4(st["wq"][r:r + step], st["ws"][r:r + step], case["k"]).t()
                          for r in range(0, case["n"], step)], 1)
    page, lens, starts = case["page"], st["lens"].tolist(), st["starts"].tolist()
    if kind == "append":
        if case["batch"] * -(-case["new"] // page) > 4096:
            return None
        out = {n: st[n].double() for n in ("k", "v")}
        table = st["table"].tolist()
        for b, length in enumerate(lens):
            at, row = length - (starts[b + 1] - starts[b]), starts[b]
            while at < length:
                p, a = table[b][at // page], at % page
                n = min(page - a, length - at)
                for name, new in (("k", st["nk"]), ("v", st["nv"])):
                    x = new[row:row + n].double().transpose(0, 1)                                # [h, n, d]
                    codes = out[name][p] if name == "k" else out[name][p].transpose(1, 2)
                    e = _least8(x.abs().amax((1, 2)))
                    if a:
                        had = st[name + "s"][p].double() - 127
                        e = torch.maximum(e, had)
                        codes[:, :a] = _nearest(codes[:, :a] * _two64(had - e)[:, None, None], 3, -6)
                    codes[:, a:a + n] = _nearest(x * _two64(-e)[:, None, None], 3, -6)
                at, row = at + n, row + n
        return {"k": out["k"], "v": out["v"], "ks": None, "vs": None}
    h, d, group = case["heads"], case["dim"], case["q_heads"] // case["heads"]
    out = torch.empty(st["q"].shape, device="cuda", dtype=torch.float64)
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        ids = st["table"][b, :-(-length // page)].long()
        k = st["k"][ids].double() * _two64(st["ks"][ids].long() - 127)[..., None, None]
        k = k.transpose(0, 1).reshape(h, -1, d)[:, :length]
        v = st["v"][ids].double() * _two64(st["vs"][ids].long() - 127)[..., None, None]
        v = v.permute(1, 0, 3, 2).reshape(h, -1, d)[:, :length]
        q = st["q"][starts[b]:starts[b + 1]].double().view(n, h, group, d)
        at = length - n + torch.arange(n, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None]
        hidden = (j > at) | ((j <= at - case["window"]) if case["window"] else False)
        for i in range(h):
            s = q[:, i].reshape(n * group, d) @ k[i].t().contiguous() / math.sqrt(d)
            s = s.view(n, group, length).masked_fill_(hidden[:, None], -math.inf)
            out[starts[b]:starts[b + 1]].view(n, h, group, d)[:, i] = torch.matmul(
                torch.softmax(s, -1).view(n * group, length), v[i]).view(n, group, d)
    return out
