"""The attention half of a decoder layer, as cases to time and to check.

Three operators around one paged key/value cache: norms and position
rotation of queries and keys (`norm_rope`), appending keys and values with
the rotation on the way (`append`), and attention of each sequence's new
tokens over its pages (`attention`).  Inputs are N(0, 1) projections (as a
packed q|k|v row per token), norm weights around 1, positions that reach
from a short prompt to a long context, and block tables that scatter a
sequence's pages over the cache.  All of it is made on the GPU from the
seed with torch alone.

With `own` the calls go to this package; without, the same results come from
elementary torch operations in 32 bits (angles in 64), rounded once.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


def _mer():
    import importlib

    return importlib.import_module("micro-expert-router-ssd-streamed-moe-mer_amd")


# ---- cases ---------------------------------------------------------------

def listed():
    return [
        # One decode token of a 32-head / 4-group model whose q and k are
        # normed per head: the smallest call, between projection and cache.
        dict(name="norm_rope_1tok", kind="norm_rope", tokens=1, heads=32, kv_heads=4, head_dim=128, rot=128,
             interleaved=False, norm=True, src="f16", dst="f16", pos=20000),
        # The same for a prompt of 4096 tokens.
        dict(name="norm_rope_4096tok", kind="norm_rope", tokens=4096, heads=32, kv_heads=4, head_dim=128, rot=128,
             interleaved=False, norm=True, src="bf16", dst="bf16", pos=8192),
        # Projections kept in f32, rotation of neighbouring pairs over a part
        # of the head, no norm, a prompt length that fits no tile.
        dict(name="rope_777tok_f32", kind="norm_rope", tokens=777, heads=32, kv_heads=8, head_dim=96, rot=64,
             interleaved=True, norm=False, src="f32", dst="f16", pos=131072),
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
        # One decode token over a short context: latency.
        dict(name="attn_decode_1x700", kind="attention", seqs=1, decode=1, q_lo=1, q_hi=1, ctx_lo=700, ctx_hi=700,
             heads=32, kv_heads=4, head_dim=128, page=16, dtype="f16", window=0, sinks=False),
        # A decode batch with ragged contexts: the serving engine's step.
        dict(name="attn_decode_64x4k", kind="attention", seqs=64, decode=64, q_lo=1, q_hi=1, ctx_lo=200, ctx_hi=8000,
             heads=32, kv_heads=8, head_dim=128, page=16, dtype="bf16", window=0, sinks=False),
        # One token over a very long context: the keys have to be split.
        dict(name="attn_decode_1x131k", kind="attention", seqs=1, decode=1, q_lo=1, q_hi=1, ctx_lo=131000,
             ctx_hi=131000, heads=32, kv_heads=8, head_dim=128, page=64, dtype="f16", window=0, sinks=False),
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
    kind = rng.choice(["norm_rope", "append", "attention", "attention", "attention"])
    d = rng.choice([64, 64, 80, 96, 112, 128, 128, 128, 128, 192, 256])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 12, 16])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    half = rng.choice(["f16", "bf16"])
    if kind != "attention":
        tokens = _logint(rng, 1, 8192)
        rot = rng.choice([d, d, d, 8 * rng.randint(1, d // 8)])
        c = dict(kind=kind, tokens=tokens, kv_heads=kv_heads, head_dim=d, rot=rot, interleaved=rng.random() < 0.3,
                 norm=rng.random() < 0.5, src=rng.choice(["f32", "f16", "bf16"]), dst=half,
                 pos=_logint(rng, 2 * tokens, 1 << 20))
        if kind == "norm_rope":
            c.update(heads=kv_heads * group, dst=rng.choice(["f32", half, half]))
            while c["tokens"] > 1 and c["tokens"] * (c["heads"] + kv_heads) * d > 4096 * 36 * 128:
                c["tokens"] = c["tokens"] * 2 // 3
            return c
        page = rng.choice([8, 16, 32, 64, 128, 256])
        c.update(page=page, pad=rng.choice([0, tokens // rng.randint(2, 9)]),
                 pages=-(-tokens // page) + rng.randint(1, 8))
        return c
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    window = rng.choice([0, 0, rng.randint(1, 4096)])
    form = rng.choice(["decode", "chunks", "mixed"])
    seqs = 1 if form == "chunks" and rng.random() < 0.5 else _logint(rng, 1, 64)
    decode = seqs if form == "decode" else 0 if form == "chunks" else rng.randint(0, seqs)
    ctx_hi = _logint(rng, 1, 65536 if seqs < 8 else 8192)
    q_hi = 1 if decode == seqs else _logint(rng, 2, 4096)
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


# ---- inputs --------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _inv_freq(rot):
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEV)
    return (1.0 / 1e6 ** (i / rot)).to(torch.float32)


def prepare(case, seed):
    g = _gen(seed)
    kind, d, kvh = case["kind"], case["head_dim"], case["kv_heads"]
    s = dict(case=case)
    if kind == "attention":
        new, keys = lengths(case)
        dt, page, h = DTYPES[case["dtype"]], case["page"], case["heads"]
        need = [-(-n // page) for n in keys]
        width, total = max(need), sum(need)
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        s["k"] = torch.randn(total, kvh, page, d, generator=g, device=DEV, dtype=dt)
        s["v"] = torch.randn(total, kvh, page, d, generator=g, device=DEV, dtype=dt)
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
        if own:
            s["cache"] = _mer().PagedKvCache.wrap(s["k"], s["v"])
        return s
    t, src = case["tokens"], DTYPES[case["src"]]
    s["inv_freq"] = _inv_freq(case["rot"])
    s["positions"] = (int(torch.randint(0, case["pos"] - t, (1,), generator=g, device=DEV))
                      + torch.arange(t, device=DEV)).to(torch.int32)
    s["k_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV) if case["norm"] else None
    if kind == "norm_rope":
        h = case["heads"]
        row = torch.randn(t, (h + 2 * kvh) * d, generator=g, device=DEV).to(src)
        s["q"] = row[:, :h * d].view(t, h, d)
        s["k"] = row[:, h * d:(h + kvh) * d].view(t, kvh, d)
        s["q_norm"] = 1.0 + 0.1 * torch.randn(d, generator=g, device=DEV) if case["norm"] else None
        return s
    row = torch.randn(t, 2 * kvh * d, generator=g, device=DEV).to(src)
    s["k"] = row[:, :kvh * d].view(t, kvh, d)
    s["v"] = row[:, kvh * d:].view(t, kvh, d)
    dst, page, pages = DTYPES[case["dst"]], case["page"], case["pages"]
    s["cache_k"] = torch.randn(pages, kvh, page, d, generator=g, device=DEV).to(dst)
    s["cache_v"] = torch.randn(pages, kvh, page, d, generator=g, device=DEV).to(dst)
    # whole pages in any order, as an allocator hands them out
    order = torch.randperm(pages, generator=g, device=DEV)
    slots = (order[:, None] * page + torch.arange(page, device=DEV)).view(-1)[:t].to(torch.int64).contiguous()
    if case["pad"]:
        slots[torch.randperm(t, generator=g, device=DEV)[:case["pad"]]] = -1
    s["slots"] = slots
    if own:
        s["cache"] = _mer().PagedKvCache.wrap(s["cache_k"], s["cache_v"])
    return s


# ---- one pass ------------------------------------------------------------

def _norm_rope(x, w, positions, inv_freq, interleaved):
    """x [t, h, d] in f32 -> normed and rotated, f32."""
    x = x.to(torch.float32)
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * w
    angle = positions.to(torch.float64)[:, None] * inv_freq.to(torch.float64)
    c, s = torch.cos(angle).to(torch.float32)[:, None], torch.sin(angle).to(torch.float32)[:, None]
    rot = 2 * inv_freq.shape[0]
    r, rest = x[:, :, :rot], x[:, :, rot:]
    if interleaved:
        a, b = r[:, :, 0::2], r[:, :, 1::2]
        r = torch.stack((a * c - b * s, b * c + a * s), 3).flatten(2)
    else:
        a, b = r[:, :, :rot // 2], r[:, :, rot // 2:]
        r = torch.cat((a * c - b * s, b * c + a * s), 2)
    return torch.cat((r, rest), 2)


def _pages(cache, table, n):
    """The first n keys (or values) of a sequence: [kv_heads, n, d]."""
    pages, kvh, page, d = cache.shape
    rows = cache[table[:-(-n // page)].to(torch.int64)]
    return rows.permute(1, 0, 2, 3).reshape(kvh, -1, d)[:, :n]


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
    if c["kind"] == "norm_rope":
        dst = DTYPES[c["dst"]]
        if own:
            return _mer().qk_norm_rope(state["q"], state["k"], state["positions"], state["inv_freq"],
                                       q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS,
                                       interleaved=c["interleaved"], out_dtype=dst)
        return tuple(_norm_rope(state[x], state[x + "_norm"], state["positions"], state["inv_freq"],
                                c["interleaved"]).to(dst) for x in ("q", "k"))
    if c["kind"] == "append":
        if own:
            _mer().kv_append(state["cache"], state["k"], state["v"], state["slots"], positions=state["positions"],
                             inv_freq=state["inv_freq"], k_norm=state["k_norm"], eps=EPS,
                             interleaved=c["interleaved"])
        else:
            k = _norm_rope(state["k"], state["k_norm"], state["positions"], state["inv_freq"], c["interleaved"])
            keep = (state["slots"] >= 0).nonzero()[:, 0]
            page, at = state["slots"][keep] // c["page"], state["slots"][keep] % c["page"]
            state["cache_k"][page, :, at] = k[keep].to(DTYPES[c["dst"]])
            state["cache_v"][page, :, at] = state["v"][keep].to(torch.float32).to(DTYPES[c["dst"]])
        return state["cache_k"], state["cache_v"]
    if own:
        return _mer().paged_attention(state["cache"], state["q"], state["table"], state["q_start"], state["kv_len"],
                                      max_q_len=max(state["new"]), max_kv_len=max(state["keys"]), window=c["window"],
                                      sinks=state["sinks"], out=state["out"])
    out = state["out"]
    for i, n in enumerate(state["keys"]):
        rows = slice(state["starts"][i], state["starts"][i + 1])
        k = _pages(state["k"], state["table"][i], n).to(torch.float32)
        v = _pages(state["v"], state["table"][i], n).to(torch.float32)
        q = state["q"][rows].to(torch.float32).transpose(0, 1).contiguous()
        out[rows] = _attention(q, k, v, c["window"], state["sinks"]).transpose(0, 1).to(out.dtype)
    return out


# ---- what a pass cannot do without ---------------------------------------

def work(case):
    kind, d, kvh = case["kind"], case["head_dim"], case["kv_heads"]
    if kind == "norm_rope":
        n = case["tokens"] * (case["heads"] + kvh) * d
        small = 4 * case["tokens"] + 2 * case["rot"] + (8 * d if case["norm"] else 0)
        return {"bytes": n * (BYTES[case["src"]] + BYTES[case["dst"]]) + small,
                "flops": n * ((4 if case["norm"] else 0) + 3)}
    if kind == "append":
        n = (case["tokens"] - case["pad"]) * kvh * d
        small = 12 * case["tokens"] + 2 * case["rot"] + (4 * d if case["norm"] else 0)
        return {"bytes": 2 * n * (BYTES[case["src"]] + BYTES[case["dst"]]) + small,
                "flops": n * ((4 if case["norm"] else 0) + 3)}
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
    return {"bytes": 4 * sum(new) * h * d + 4 * read * kvh * d + 4 * read // case["page"],
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


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm_rope":
        return tuple(_rotate64(s[x].clone(), s[x + "_norm"], s["positions"], s["inv_freq"], case["interleaved"])
                     for x in ("q", "k"))
    if case["kind"] == "append":
        k = _rotate64(s["k"].clone(), s["k_norm"], s["positions"], s["inv_freq"], case["interleaved"])
        outs = []
        for cache, rows in ((s["cache_k"], k), (s["cache_v"], s["v"].to(torch.float64))):
            flat = cache.to(torch.float64).transpose(1, 2).contiguous()  # [pages, page, heads, d]
            flat = flat.view(-1, *flat.shape[2:])
            put = s["slots"] >= 0
            flat[s["slots"][put]] = rows[put]
            outs.append(flat.view(case["pages"], case["page"], *flat.shape[1:]).transpose(1, 2).contiguous())
        return tuple(outs)
    # row by row groups: every head's keys and values gathered one by one
    group, d, w = case["heads"] // case["kv_heads"], case["head_dim"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, (n, l) in enumerate(zip(s["new"], s["keys"])):
        j = torch.arange(l, device=DEV)
        page, at = s["table"][i, j // case["page"]].to(torch.int64), j % case["page"]
        for g in range(case["kv_heads"]):
            k, v = s["k"][page, g, at].to(torch.float64), s["v"][page, g, at].to(torch.float64)
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
