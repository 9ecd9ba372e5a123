"""A paged key/value cache held in 4 bits, as cases to time and to check.

Three operators around it: appending keys and values, quantised as they are
written with the key's norm and rotation on the way (`append`, which also
reads the pages back that it wrote to), reading rows back (`read`), and
attention of each sequence's new tokens over the cache (`attention`).

A block is 32 neighbouring elements of a head.  Its scale d is that of the
element a of largest magnitude (the positive one of two equal ones): |a| / 8
rounded to five bits, held as float16 with the sign opposite to a's; its
codes are n = round(x / d) + 8 within 0 .. 15 and stand for d (n - 8), which
five bits of scale make exact in float16 and bfloat16 alike.  Codes lie as
[pages, kv heads, page size, head_dim / 2] bytes, a block's 16 bytes holding
elements 0 .. 15 in their low and 16 .. 31 in their high halves; scales as
[pages, kv heads, head_dim / 32, page size].

Inputs are N(0, 1) projections (as a packed row per token), norm weights
around 1, positions that reach from a short prompt to a long context, and
block tables that scatter a sequence's pages over the cache.  All of it is
made on the GPU from the seed with torch alone.

With `own` the calls go to this package; without, the same results come from
elementary torch operations in 32 bits, rounded once; keys on their way to
the cache, which lie next to a code's border now and then, are normed and
rotated in 64.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6
BLOCK = 32
D_MOST = 7936.0  # the largest scale of five bits whose eightfold is a float16


def _mer():
    import importlib

    return importlib.import_module("micro-expert-router-ssd-streamed-moe-mer_amd")


# ---- cases ---------------------------------------------------------------

def listed():
    return [
        # A decode batch: one new token of 48 sequences into their pages.
        dict(name="append_48tok", kind="append", tokens=48, pad=0, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, norm=False, page=16, pages=1024, src="f16", dst="f16", pos=16384),
        # A prompt into the cache, keys normed and rotated on the way, f32
        # projections.
        dict(name="append_4096tok_norm", kind="append", tokens=4096, pad=0, kv_heads=8, head_dim=128, rot=128,
             interleaved=False, norm=True, page=64, pages=80, src="f32", dst="bf16", pos=8192),
        # A padded batch (rows without a slot are skipped), small heads.
        dict(name="append_1000tok_pad", kind="append", tokens=1000, pad=123, kv_heads=4, head_dim=64, rot=64,
             interleaved=True, norm=False, page=32, pages=64, src="bf16", dst="bf16", pos=65536),
        # A short prefix that another sequence goes on with, back as rows.
        dict(name="read_200rows", kind="read", tokens=200, pad=9, kv_heads=8, head_dim=128, page=16, pages=512,
             dst="f16"),
        # A long context brought back for a path that works on float16 rows.
        dict(name="read_32768rows", kind="read", tokens=32768, pad=0, kv_heads=8, head_dim=128, page=64, pages=520,
             dst="bf16"),
        # One decode token over a short context: latency.
        dict(name="attn_decode_1x700", kind="attention", seqs=1, decode=1, q_lo=1, q_hi=1, ctx_lo=700, ctx_hi=700,
             heads=32, kv_heads=4, head_dim=128, page=16, dtype="f16", window=0, sinks=False),
        # A decode batch with ragged contexts: the serving engine's step.
        dict(name="attn_decode_64x4k", kind="attention", seqs=64, decode=64, q_lo=1, q_hi=1, ctx_lo=200, ctx_hi=8000,
             heads=32, kv_heads=8, head_dim=128, page=16, dtype="bf16", window=0, sinks=False),
        # One token over a very long context: the keys have to be split.
        dict(name="attn_decode_1x131k", kind="attention", seqs=1, decode=1, q_lo=1, q_hi=1, ctx_lo=131000,
             ctx_hi=131000, heads=32, kv_heads=8, head_dim=128, page=64, dtype="f16", window=0, sinks=False),
        # Five tokens of sixteen sequences (a draft to be checked), 25 rows to
        # a kv head, heads that fill no power of two.
        dict(name="attn_draft_16x5", kind="attention", seqs=16, decode=0, q_lo=5, q_hi=5, ctx_lo=2000, ctx_hi=6000,
             heads=40, kv_heads=8, head_dim=96, page=32, dtype="f16", window=0, sinks=False),
        # A whole prompt of 4096 tokens: the largest rate.
        dict(name="attn_prompt_4096", kind="attention", seqs=1, decode=0, q_lo=4096, q_hi=4096, ctx_lo=0, ctx_hi=0,
             heads=32, kv_heads=8, head_dim=128, page=64, dtype="bf16", window=0, sinks=False),
        # A chunk of a long prompt over what is in the cache already, beside
        # another sequence's chunk; eight heads to a group.
        dict(name="attn_chunk_512_of_32k", kind="attention", seqs=2, decode=0, q_lo=400, q_hi=640, ctx_lo=20000,
             ctx_hi=36000, heads=32, kv_heads=4, head_dim=128, page=32, dtype="f16", window=0, sinks=False),
        # A mixed batch: 24 decoding sequences and 8 chunks in one call,
        # sliding window and a sink per head, heads of 64.
        dict(name="attn_mixed_window", kind="attention", seqs=32, decode=24, q_lo=33, q_hi=500, ctx_lo=0, ctx_hi=5000,
             heads=64, kv_heads=8, head_dim=64, page=16, dtype="bf16", window=1024, sinks=True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attention", "attention", "attention", "attention"])
    d = rng.choice([32, 64, 64, 96, 128, 128, 128, 128, 160, 192, 224, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    half = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if kind != "attention":
        tokens = _logint(rng, 1, 8192 if kind == "append" else 32768)
        while tokens > 1 and tokens * kv_heads * d > (1 << 23 if kind == "append" else 1 << 25):
            tokens = tokens * 2 // 3
        c = dict(kind=kind, tokens=tokens, kv_heads=kv_heads, head_dim=d, page=page,
                 pad=rng.choice([0, tokens // rng.randint(2, 9)]), pages=-(-tokens // page) + rng.randint(1, 8), dst=half)
        if kind == "read":
            return c
        c.update(rot=rng.choice([d, d, d, 8 * rng.randint(1, d // 8)]), interleaved=rng.random() < 0.3,
                 norm=rng.random() < 0.5, src=rng.choice(["f32", "f16", "bf16"]), pos=_logint(rng, 2 * tokens, 1 << 20))
        return c
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16])
    window = rng.choice([0, 0, rng.randint(1, 4096)])
    form = rng.choice(["decode", "draft", "chunks", "mixed"])
    seqs = 1 if form == "chunks" and rng.random() < 0.5 else _logint(rng, 1, 64)
    decode = seqs if form == "decode" else 0 if form in ("draft", "chunks") else rng.randint(0, seqs)
    ctx_hi = _logint(rng, 1, 65536 if seqs < 8 else 8192)
    q_hi = 1 if decode == seqs else rng.randint(2, 8) if form == "draft" else _logint(rng, 2, 4096)
    while q_hi > 2 and (seqs - decode) * q_hi * (ctx_hi + q_hi) > 1 << 25:
        q_hi = q_hi * 2 // 3
    while ctx_hi > 2 and ((seqs - decode) * q_hi * (ctx_hi + q_hi) * kv_heads * group * d > 1 << 36
                          or seqs * ctx_hi * kv_heads * d > 1 << 28):
        ctx_hi = ctx_hi * 2 // 3
        q_hi = max(min(q_hi, 2), q_hi * 5 // 6)
    return dict(kind=kind, seqs=seqs, decode=decode, q_lo=rng.randint(1, q_hi), q_hi=q_hi,
                ctx_lo=rng.randint(0, ctx_hi), ctx_hi=ctx_hi, heads=kv_heads * group, kv_heads=kv_heads, head_dim=d,
                page=page, dtype=half, window=window, sinks=rng.random() < 0.3)


def _spread(i, lo, hi, phase):
    """The i-th length between lo and hi: evenly spread, in no order."""
    return lo + int((hi - lo + 1) * math.fmod((i + phase) * 0.6180339887498949, 1.0))


def lengths(case):
    """(new tokens, keys with the new ones) of every sequence."""
    new = [1 if i < case["decode"] else _spread(i, case["q_lo"], case["q_hi"], 0.5) for i in range(case["seqs"])]
    return new, [n + _spread(i, case["ctx_lo"], case["ctx_hi"], 0.25) for i, n in enumerate(new)]


# ---- the 4-bit form ------------------------------------------------------

def _quantise(x):
    """x [..., d] in f32 -> (codes [..., d / 2], scales [..., d / 32] f16)."""
    x = x.unflatten(-1, (-1, BLOCK))
    hi, lo = x.amax(-1), x.amin(-1)
    a = torch.where(hi >= -lo, hi, lo)
    m, e = torch.frexp(a.abs() / 8)
    d = torch.ldexp(torch.round(m * 32), e - 5).to(torch.float16).clamp(max=D_MOST)
    d = torch.where(a > 0, -d, d)
    dd = d.to(torch.float32)[..., None]
    n = torch.where(dd == 0, 0.0, torch.round(x / dd)).clamp(-8, 7) + 8
    n = n.to(torch.uint8)
    return (n[..., :16] | n[..., 16:] << 4).flatten(-2), d


def _values(codes, scales):
    """The f32 values of codes [..., d / 2] with scales [..., d / 32]."""
    b = codes.unflatten(-1, (-1, BLOCK // 2))
    n = torch.cat((b & 15, b >> 4), -1).to(torch.float32) - 8
    return (n * scales.to(torch.float32)[..., None]).flatten(-2)


# ---- inputs --------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inv_freq(rot):
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEV)
    return (1.0 / 1e6 ** (i / rot)).to(torch.float32)


def _cache(s, pages, kvh, page, d, g):
    """Pages of N(0, 1) keys and values, some million at a time."""
    for x in ("k", "v"):
        codes = torch.empty(pages, kvh, page, d // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(pages, kvh, d // BLOCK, page, dtype=torch.float16, device=DEV)
        step = max(1, (1 << 25) // (kvh * page * d))
        for a in range(0, pages, step):
            b = min(pages, a + step)
            c, sc = _quantise(torch.randn(b - a, kvh, page, d, generator=g, device=DEV))
            codes[a:b] = c
            scales[a:b] = sc.transpose(2, 3)
        s[x + "_codes"], s[x + "_scales"] = codes, scales
    if own:
        s["cache"] = _mer().PagedKvCacheQ4.wrap(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])


def prepare(case, seed):
    g = _gen(seed)
    kind, d, kvh, page = case["kind"], case["head_dim"], case["kv_heads"], case["page"]
    s = dict(case=case)
    if kind == "attention":
        new, keys = lengths(case)
        dt, h = DTYPES[case["dtype"]], case["heads"]
        need = [-(-n // page) for n in keys]
        width, total = max(need), sum(need)
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        _cache(s, total, kvh, page, d, g)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        # q and k of trained models agree more than chance: logits of spread 2
        s["q"] = (2.0 * torch.randn(starts[-1], h, d, generator=g, device=DEV)).to(dt)
        s["table"], s["new"], s["keys"], s["starts"] = table, new, keys, starts
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["kv_len"] = torch.tensor(keys, dtype=torch.int32, device=DEV)
        s["sinks"] = torch.randn(h, generator=g, device=DEV) if case["sinks"] else None
        s["out"] = torch.empty_like(s["q"])
        return s
    t, pages = case["tokens"], case["pages"]
    _cache(s, pages, kvh, page, d, g)
    # whole pages in any order, as an allocator hands them out
    order = torch.randperm(pages, generator=g, device=DEV)
    places = (order[:, None] * page + torch.arange(page, device=DEV)).view(-1).to(torch.int64)
    slots = places[:t].clone()
    if case["pad"]:
        slots[torch.randperm(t, generator=g, device=DEV)[:case["pad"]]] = -1
    s["slots"] = slots
    dst = DTYPES[case["dst"]]
    if kind == "append":
        row = torch.randn(t, 2 * kvh * d, generator=g, device=DEV).to(DTYPES[case["src"]])
        s["k"] = row[:, :kvh * d].view(t, kvh, d)
        s["v"] = row[:, kvh * d:].view(t, kvh, d)
        s["inv_freq"] = _inv_freq(case["rot"])
        s["positions"] = (int(torch.randint(0, case["pos"] - t, (1,), generator=g, device=DEV))
                          + torch.arange(t, device=DEV)).to(torch.int32)
        s["k_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV) if case["norm"] else None
        # every place of the pages that rows go to
        slots = places[:-(-t // page) * page].contiguous()
    s["back"] = slots
    s["k_out"] = torch.empty(slots.numel(), kvh, d, dtype=dst, device=DEV)
    s["v_out"] = torch.empty(slots.numel(), kvh, d, dtype=dst, device=DEV)
    return s


# ---- one pass ------------------------------------------------------------

def _norm_rope(x, w, positions, inv_freq, interleaved):
    """x [t, h, d] -> normed and rotated in 64 bits, as f32."""
    x = x.to(torch.float64)
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * w.to(torch.float64)
    angle = positions.to(torch.float64)[:, None] * inv_freq.to(torch.float64)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    rot = 2 * inv_freq.shape[0]
    r, rest = x[:, :, :rot], x[:, :, rot:]
    if interleaved:
        a, b = r[:, :, 0::2], r[:, :, 1::2]
        r = torch.stack((a * c - b * s, b * c + a * s), 3).flatten(2)
    else:
        a, b = r[:, :, :rot // 2], r[:, :, rot // 2:]
        r = torch.cat((a * c - b * s, b * c + a * s), 2)
    return torch.cat((r, rest), 2).to(torch.float32)


def _read(state, x):
    """The rows state["back"] of the keys or values; zeros for padding."""
    slots, page = state["back"], state["case"]["page"]
    at, place = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    y = _values(state[x + "_codes"][at, :, place], state[x + "_scales"][at, :, :, place])
    return torch.where((slots >= 0)[:, None, None], y, 0.0)


def _pages(state, x, i, n):
    """The first n keys (or values) of sequence i: [kv_heads, n, d]."""
    codes, scales = state[x + "_codes"], state[x + "_scales"]
    rows = state["table"][i, :-(-n // codes.shape[2])].to(torch.int64)
    y = _values(codes[rows], scales[rows].transpose(2, 3))
    return y.permute(1, 0, 2, 3).reshape(codes.shape[1], -1, y.shape[3])[:, :n]


def _attention(q, k, v, window, sinks):
    """q [h, n, d], k and v [kv_heads, l, d] in f32; the n rows are the last
    positions of the l keys."""
    h, n, d = q.shape
    kvh, l, _ = k.shape
    out = torch.empty_like(q)
    for a in range(0, n, 1024):  # rows in pieces, so the scores stay small
        b = min(n, a + 1024)
        pos = torch.arange(l - n + a, l - n + b, device=q.device)
        lo, hi = (0 if window == 0 else max(0, l - n + a - window + 1)), l - n + b
        j = torch.arange(lo, hi, device=q.device)
        seen = j <= pos[:, None]
        if window:
            seen &= j > pos[:, None] - window
        qq = q[:, a:b].reshape(kvh, -1, d)
        s = torch.matmul(qq, k[:, lo:hi].transpose(1, 2).contiguous()) * d ** -0.5
        s = torch.where(seen, s.view(h, b - a, -1), -math.inf)
        m = s.amax(2, keepdim=True)
        if sinks is not None:
            m = torch.maximum(m, sinks[:, None, None])
        p = torch.exp(s - m)
        z = p.sum(2, keepdim=True)
        if sinks is not None:
            z = z + torch.exp(sinks[:, None, None] - m)
        o = torch.matmul(p.view(kvh, -1, hi - lo), v[:, lo:hi].contiguous())
        out[:, a:b] = o.view(h, b - a, d) / z
    return out


def run(state):
    c = state["case"]
    if c["kind"] == "append":
        if own:
            _mer().kv_append(state["cache"], state["k"], state["v"], state["slots"], positions=state["positions"],
                             inv_freq=state["inv_freq"], k_norm=state["k_norm"], eps=EPS,
                             interleaved=c["interleaved"])
        else:
            k = _norm_rope(state["k"], state["k_norm"], state["positions"], state["inv_freq"], c["interleaved"])
            keep = (state["slots"] >= 0).nonzero()[:, 0]
            page, at = state["slots"][keep] // c["page"], state["slots"][keep] % c["page"]
            for x, y in (("k", k), ("v", state["v"].to(torch.float32))):
                codes, scales = _quantise(y[keep])
                state[x + "_codes"][page, :, at] = codes
                state[x + "_scales"][page, :, :, at] = scales
    if c["kind"] != "attention":
        if own:
            return _mer().kv_read(state["cache"], state["back"], k_out=state["k_out"], v_out=state["v_out"])
        state["k_out"].copy_(_read(state, "k"))
        state["v_out"].copy_(_read(state, "v"))
        return state["k_out"], state["v_out"]
    if own:
        return _mer().paged_attention(state["cache"], state["q"], state["table"], state["q_start"], state["kv_len"],
                                      max_q_len=max(state["new"]), max_kv_len=max(state["keys"]), window=c["window"],
                                      sinks=state["sinks"], out=state["out"])
    out = state["out"]
    for i, n in enumerate(state["keys"]):
        rows = slice(state["starts"][i], state["starts"][i + 1])
        q = state["q"][rows].to(torch.float32).transpose(0, 1).contiguous()
        o = _attention(q, _pages(state, "k", i, n), _pages(state, "v", i, n), c["window"], state["sinks"])
        out[rows] = o.transpose(0, 1).to(out.dtype)
    return out


# ---- what a pass cannot do without ---------------------------------------

def work(case):
    kind, d, kvh = case["kind"], case["head_dim"], case["kv_heads"]
    held = d // 2 + d // 16  # bytes of a head's key or value in the cache
    if kind == "read":
        n, t = (case["tokens"] - case["pad"]) * kvh, case["tokens"] * kvh
        return {"bytes": 2 * n * held + 2 * t * d * BYTES[case["dst"]] + 8 * case["tokens"], "flops": 4 * n * d}
    if kind == "append":
        n = (case["tokens"] - case["pad"]) * kvh
        back = -(-case["tokens"] // case["page"]) * case["page"]
        small = 12 * case["tokens"] + 8 * back + 2 * case["rot"] + (4 * d if case["norm"] else 0)
        return {"bytes": 2 * n * (d * BYTES[case["src"]] + held) + 2 * back * kvh * (d * BYTES[case["dst"]] + held) + small,
                "flops": n * d * ((4 if case["norm"] else 0) + 3 + 2 * 4) + 4 * back * kvh * d}
    new, keys = lengths(case)
    w = case["window"]
    read = pairs = 0
    for n, l in zip(new, keys):
        first = l - n
        read += l - (max(0, first - w + 1) if w else 0)
        if w:
            short = max(0, min(l, w) - first)  # rows that the window does not cut
            pairs += short * first + short * (short + 1) // 2 + (n - short) * w
        else:
            pairs += n * first + n * (n + 1) // 2
    h = case["heads"]
    return {"bytes": 4 * sum(new) * h * d + 2 * read * kvh * held + 4 * read // case["page"],
            "flops": 4 * pairs * h * d}


# ---- the same in 64 bits -------------------------------------------------

def _rotate64(x, w, positions, inv_freq, interleaved):
    y = x.to(torch.float64)
    if w is not None:
        y = y / torch.sqrt(torch.mean(y ** 2, dim=-1, keepdim=True) + EPS) * w.to(torch.float64)
    half = inv_freq.shape[0]
    i = torch.arange(half, device=y.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=y.device),
                       torch.outer(positions.to(torch.float64), inv_freq.to(torch.float64)))
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _held64(y):
    """What a cache holds of y (f64, meant as f32): by comparing with borders."""
    y = y.to(torch.float32).to(torch.float64)
    out = torch.empty_like(y)
    for b in range(0, y.shape[-1], BLOCK):
        x = y[..., b:b + BLOCK]
        most = x.abs().amax(-1, keepdim=True)
        top = (x == most).any(-1, keepdim=True)  # a positive one is among the largest
        bits = (most / 8).to(torch.float32).view(torch.int32)
        bits = (bits + 0x3ffff + (bits >> 19 & 1)) & ~0x7ffff  # four bits behind the first
        d = bits.view(torch.float32).to(torch.float16).to(torch.float64).clamp(max=D_MOST)
        d = torch.where(top, -d, d)
        t = torch.where(d == 0, 0.0, x / torch.where(d == 0, 1.0, d))
        n = torch.floor(t)
        rest = t - n
        n = n + ((rest > 0.5) | ((rest == 0.5) & (n % 2 == 1)))
        out[..., b:b + BLOCK] = n.clamp(-8, 7) * d
    return out


def _at64(s, x, page, head, place):
    """Elements [.., d] of places of pages, one code at a time."""
    codes, scales = s[x + "_codes"][page, head, place], s[x + "_scales"][page, head, :, place]
    i = torch.arange(2 * codes.shape[-1], device=codes.device)
    byte = codes[..., i // BLOCK * (BLOCK // 2) + i % 16].to(torch.int32)
    n = torch.where(i % BLOCK < 16, byte & 15, byte >> 4)
    return (n - 8).to(torch.float64) * scales[..., i // BLOCK].to(torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "attention":
        outs, slots, page = [], s["back"], case["page"]
        there = (slots >= 0)[:, None]
        for x in ("k", "v"):
            at, place = slots.clamp(min=0) // page, slots.clamp(min=0) % page
            rows = torch.stack([torch.where(there, _at64(s, x, at, g, place), 0.0) for g in range(case["kv_heads"])], 1)
            if case["kind"] == "append":
                y = s["v"].to(torch.float64) if x == "v" else _rotate64(
                    s["k"].clone(), s["k_norm"], s["positions"], s["inv_freq"], case["interleaved"])
                # the rows appended stand first among those read back, in their order
                put = (s["slots"] >= 0).nonzero()[:, 0]
                rows[put] = _held64(y[put])
            outs.append(rows)
        return tuple(outs)
    # row by row groups: every head's keys and values gathered one by one
    group, d, w = case["heads"] // case["kv_heads"], case["head_dim"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, (n, l) in enumerate(zip(s["new"], s["keys"])):
        j = torch.arange(l, device=DEV)
        page, at = s["table"][i, j // case["page"]].to(torch.int64), j % case["page"]
        for g in range(case["kv_heads"]):
            k, v = _at64(s, "k", page, g, at), _at64(s, "v", page, g, at)
            for a in range(0, n, 512):
                b = min(n, a + 512)
                p = l - n + torch.arange(a, b, device=DEV)[:, None]
                hide = (j > p) | ((j + w <= p) if w else torch.zeros_like(j > p))
                for h in range(g * group, (g + 1) * group):
                    rows = slice(s["starts"][i] + a, s["starts"][i] + b)
                    logit = s["q"][rows, h].to(torch.float64) @ k.T / math.sqrt(d)
                    logit.masked_fill_(hide, -math.inf)
                    if s["sinks"] is not None:
                        logit = torch.cat((logit, s["sinks"][h].to(torch.float64).expand(b - a, 1)), 1)
                    out[rows, h] = torch.softmax(logit, 1)[:, :l] @ v
    return out
