"""Norm and rotation of q and k, append to a paged cache, attention over it:
each against its formula in 64 bits on the CPU.

Tolerances count roundings (half a step of a type t relative to a value is
finfo(t).eps / 2 = h):
  - norm and rotation compute in f32 and round once to the output type.  A
    norm's factor and two products are within 16 f32 half steps of the exact
    ones (a sum of head_dim / 8 + 3 terms deep <= 35 additions of positive
    terms enters through a square root: 18 half steps; division, root and
    three products: 6 more), a turned element adds an angle error of 2^-24 of
    a turn (2 pi 2^-24 rad) and the sine's own few half steps, relative to the
    pair's length.  48 f32 half steps of the pair's length cover both:
    |got - want| <= h_out |want| + 48 h_f32 |pair|.
  - attention rounds P to the cache's type (h each), so the output is off by
    at most h sum_j p_j |v_j| / sum_j p_j, and the scores' f32 error
    (head_dim products of exact 16-bit factors: <= (head_dim / 16 + 8) half
    steps of sum |q_d k_d| scale, entering the exponent) moves each weight
    by that much, relatively; twice that with the sum below the fraction; then
    one rounding of the output.
"""
from __future__ import annotations

import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# ---- formulas in 64 bits -------------------------------------------------

def norm_rope64(x, w, positions, inv_freq, eps, interleaved):
    """(result, length of each element's pair) of x [t, h, d]."""
    y = x.to(torch.float64)
    if w is not None:
        y = y / (y.pow(2).mean(2, keepdim=True) + eps).sqrt() * w.to(torch.float64)
    size = y.abs()
    if inv_freq is None:
        return y, size
    out, half = y.clone(), inv_freq.numel()
    a = positions.to(torch.float64)[:, None] * inv_freq.to(torch.float64)
    c, s = a.cos()[:, None], a.sin()[:, None]
    i = torch.arange(half)
    u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out[..., u] = y[..., u] * c - y[..., v] * s
    out[..., v] = y[..., v] * c + y[..., u] * s
    size[..., u] = size[..., v] = (y[..., u] ** 2 + y[..., v] ** 2).sqrt()
    return out, size


def close_rope(got, want, size):
    bound = HALF[got.dtype] * want.abs() + 48 * HALF[F32] * size + 1e-30
    if got.dtype == F16:
        bound = bound + 2.0 ** -25  # half a step of its subnormals
    err = (got.cpu().to(torch.float64) - want).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst} of the bound"


def attention64(q, k, v, first, window, sinks, scale, h):
    """One sequence: q [n, H, d], k and v [L, G, d] in float64; row i stands at
    first + i.  Returns (out, bound) with the rounding bound above."""
    n, heads, d = q.shape
    keys, groups, _ = k.shape
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    j, p = torch.arange(keys), first + torch.arange(n)[:, None]
    seen = j <= p
    if window:
        seen &= j > p - window
    for hd in range(heads):
        g = hd // (heads // groups)
        kk, vv, qq = k[:, g], v[:, g], q[:, hd]
        s = torch.where(seen, qq @ kk.T * scale, -math.inf)
        size = torch.where(seen, qq.abs() @ kk.abs().T * abs(scale), 0.0)
        m = s.amax(1, keepdim=True) if keys else torch.full((n, 1), -math.inf, dtype=torch.float64)
        if sinks is not None:
            m = m.clamp(min=float(sinks[hd]))
        m = torch.where(m == -math.inf, 0.0, m)
        e = torch.exp(s - m)
        z = e.sum(1, keepdim=True)
        if sinks is not None:
            z = z + torch.exp(float(sinks[hd]) - m)
        ok = z > 0
        z = torch.where(ok, z, 1.0)
        out[:, hd] = e @ vv / z
        weight = h + 2 * (d / 16 + 8) * HALF[F32] * size + 64 * HALF[F32]
        bound[:, hd] = (e * weight) @ vv.abs() / z
    return out, bound + h * out.abs()


# ---- q / k norm and rotation ---------------------------------------------

def inv_freq(rot, base=1e6):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).to(F32)


@pytest.mark.parametrize("src,dst", list(itertools.product([F32, F16, BF16], [F32, F16, BF16])))
@pytest.mark.parametrize("tokens,heads,kv,d,rot,interleaved,normed", [
    (1, 32, 4, 128, 128, False, True),
    (5, 7, 3, 64, 64, True, True),
    (37, 3, 1, 80, 40, False, False),
    (130, 12, 2, 96, 8, True, False),
    (67, 5, 5, 256, 256, False, True),
    (33, 1, 1, 8, 8, False, True),
    (9, 4, 2, 72, 72, False, True),
    (300, 16, 2, 192, 64, True, True),
])
def test_norm_rope(mer, gpu, src, dst, tokens, heads, kv, d, rot, interleaved, normed):
    g = torch.Generator().manual_seed(tokens * d + heads)
    row = torch.randn(tokens, (heads + 2 * kv) * d, generator=g).to(src)
    q, k = row[:, :heads * d].view(tokens, heads, d), row[:, heads * d:(heads + kv) * d].view(tokens, kv, d)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, dtype=torch.int32)
    pos[0] = 0
    f = inv_freq(rot)
    qn = 1 + 0.1 * torch.randn(d, generator=g) if normed else None
    kn = 1 + 0.1 * torch.randn(d, generator=g) if normed else None
    dev = row.to(gpu)
    up = lambda t: None if t is None else t.to(gpu)
    qo, ko = mer.qk_norm_rope(dev[:, :heads * d].view(tokens, heads, d),
                              dev[:, heads * d:(heads + kv) * d].view(tokens, kv, d), up(pos), up(f), q_norm=up(qn),
                              k_norm=up(kn), eps=1e-5, interleaved=interleaved, out_dtype=dst)
    for got, x, w in ((qo, q, qn), (ko, k, kn)):
        assert got.dtype == dst and got.shape == x.shape
        close_rope(got, *norm_rope64(x, w, pos, f, 1e-5, interleaved))


def test_norm_rope_parts(mer, gpu):
    """Only queries; only one norm; no rotation; negative and far positions; no tokens."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(11, 4, 64, generator=g), torch.randn(11, 2, 64, generator=g)
    w = 1 + 0.1 * torch.randn(64, generator=g)
    f = inv_freq(64)
    pos = torch.tensor([0, 1, -1, -77, 2 ** 31 - 1, -2 ** 31, 5, 6, 7, 8, 123456789], dtype=torch.int32)
    d = lambda t: t.to(gpu)
    qo, none = mer.qk_norm_rope(d(q), None, d(pos), d(f), q_norm=d(w))
    assert none is None
    close_rope(qo, *norm_rope64(q, w, pos, f, 1e-6, False))
    qo, ko = mer.qk_norm_rope(d(q), d(k), d(pos), d(f), k_norm=d(w), interleaved=True)
    close_rope(qo, *norm_rope64(q, None, pos, f, 1e-6, True))
    close_rope(ko, *norm_rope64(k, w, pos, f, 1e-6, True))
    qo, ko = mer.qk_norm_rope(d(q), d(k), None, None, q_norm=d(w), k_norm=d(w))
    close_rope(qo, *norm_rope64(q, w, None, None, 1e-6, False))
    close_rope(ko, *norm_rope64(k, w, None, None, 1e-6, False))
    qo, ko = mer.qk_norm_rope(d(q)[:0], d(k)[:0], d(pos)[:0], d(f))
    assert qo.shape == (0, 4, 64) and ko.shape == (0, 2, 64)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_norm_rope_in_place(mer, gpu, dt):
    """q and k turned where they lie in a packed q|k|v row; v and the gap after it stay."""
    g = torch.Generator().manual_seed(2)
    t, h, kv, d = 50, 6, 2, 128
    row = torch.randn(t, (h + 2 * kv) * d + 16, generator=g).to(dt)
    dev = row.to(gpu)
    q, k = dev[:, :h * d].unflatten(1, (h, d)), dev[:, h * d:(h + kv) * d].unflatten(1, (kv, d))
    pos, f = torch.arange(1000, 1000 + t, dtype=torch.int32), inv_freq(d)
    w = 1 + 0.1 * torch.randn(d, generator=g)
    mer.qk_norm_rope(q, k, pos.to(gpu), f.to(gpu), q_norm=w.to(gpu), k_norm=w.to(gpu), q_out=q, k_out=k)
    got = dev.cpu()
    assert torch.equal(got[:, (h + kv) * d:], row[:, (h + kv) * d:])
    close_rope(got[:, :h * d].unflatten(1, (h, d)), *norm_rope64(row[:, :h * d].unflatten(1, (h, d)), w, pos, f, 1e-6, False))
    close_rope(got[:, h * d:(h + kv) * d].unflatten(1, (kv, d)),
               *norm_rope64(row[:, h * d:(h + kv) * d].unflatten(1, (kv, d)), w, pos, f, 1e-6, False))


# ---- append --------------------------------------------------------------

@pytest.mark.parametrize("src,dst", list(itertools.product([F32, F16, BF16], [F16, BF16])))
@pytest.mark.parametrize("tokens,kv,d,page,rot,normed", [
    (1, 8, 128, 16, 128, False), (45, 3, 64, 8, 64, True), (129, 2, 112, 32, 0, False), (70, 1, 256, 256, 128, True),
])
def test_append(mer, gpu, src, dst, tokens, kv, d, page, rot, normed):
    g = torch.Generator().manual_seed(tokens + d)
    k = torch.randn(tokens, kv, d, generator=g).to(src)
    v = torch.randn(tokens, kv, d, generator=g).to(src)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 1:
        slots[::7] = -1
    ck = torch.full((pages, kv, page, d), 3.5, dtype=dst)
    cv = torch.full((pages, kv, page, d), -2.5, dtype=dst)
    pos = torch.randint(0, 100000, (tokens,), generator=g, dtype=torch.int32)
    f = inv_freq(rot) if rot else None
    w = 1 + 0.1 * torch.randn(d, generator=g) if normed else None
    up = lambda t: None if t is None else t.to(gpu)
    cache = mer.PagedKvCache.wrap(ck.to(gpu), cv.to(gpu))
    mer.kv_append(cache, up(k), up(v), up(slots), positions=up(pos) if rot else None, inv_freq=up(f), k_norm=up(w))
    want, size = norm_rope64(k, w, pos, f, 1e-6, False)
    gk, gv = cache.k.cpu(), cache.v.cpu()
    written = torch.zeros(pages, page, dtype=torch.bool)
    for t in range(tokens):
        if slots[t] < 0:
            continue
        pg, at = int(slots[t]) // page, int(slots[t]) % page
        written[pg, at] = True
        close_rope(gk[pg, :, at], want[t], size[t])
        assert torch.equal(gv[pg, :, at], v[t].to(dst))
    assert (gk.transpose(1, 2)[~written] == 3.5).all() and (gv.transpose(1, 2)[~written] == -2.5).all()


def test_append_past_the_cache(mer, gpu):
    mer.take_device_status()
    cache = mer.PagedKvCache.wrap(torch.zeros(2, 1, 8, 16, dtype=F16, device=gpu),
                                  torch.zeros(2, 1, 8, 16, dtype=F16, device=gpu))
    k = torch.ones(3, 1, 16, dtype=F16, device=gpu)
    mer.kv_append(cache, k, k, torch.tensor([3, 16, 1 << 40], device=gpu))
    with pytest.raises(mer.GpuExpertDispatchError):
        mer.take_device_status()
    assert cache.k.sum().item() == 16 and cache.v.sum().item() == 16


# ---- attention -----------------------------------------------------------

class Batch:
    """Sequences of (new tokens, keys) with pages in random order, NaN in every
    place that no sequence has written, page ids of -1 behind each row's pages."""

    def __init__(self, seqs, heads, kv, d, page, dt, seed, spare=3, gap=0, kscale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.page, self.dt = seqs, page, dt
        need = [-(-max(l, 0) // page) for _, l in seqs]
        width = max(need + [1]) + 1
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).to(torch.int32)
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        self.k = torch.full((total, kv, page, d), math.nan, dtype=dt)
        self.v = torch.full((total, kv, page, d), math.nan, dtype=dt)
        self.kk, self.vv, self.start = [], [], [0]
        at = 0
        for i, (n, l) in enumerate(seqs):
            ids = order[at:at + need[i]]
            at += need[i]
            self.table[i, :need[i]] = ids
            kk = (kscale * torch.randn(max(l, 0), kv, d, generator=g)).to(dt)
            vv = torch.randn(max(l, 0), kv, d, generator=g).to(dt)
            for j in range(need[i]):
                part = slice(j * page, min((j + 1) * page, l))
                m = part.stop - part.start
                self.k[ids[j], :, :m] = kk[part].transpose(0, 1)
                self.v[ids[j], :, :m] = vv[part].transpose(0, 1)
            self.kk.append(kk)
            self.vv.append(vv)
            self.start.append(self.start[-1] + n)
        self.n = self.start[-1] + gap
        self.q = torch.randn(self.n, heads, d, generator=g).to(dt)

    def run(self, mer, gpu, hints=True, **kw):
        cache = mer.PagedKvCache.wrap(self.k.to(gpu), self.v.to(gpu))
        out = torch.full_like(self.q, 7.0, device=gpu)
        more = dict(max_q_len=max(n for n, _ in self.seqs), max_kv_len=max(l for _, l in self.seqs)) if hints else {}
        more.update(kw)
        if more.get("sinks") is not None:
            more["sinks"] = more["sinks"].to(gpu)
        return mer.paged_attention(cache, self.q.to(gpu), self.table.to(gpu),
                                   torch.tensor(self.start, dtype=torch.int32, device=gpu),
                                   torch.tensor([l for _, l in self.seqs], dtype=torch.int32, device=gpu), out=out,
                                   **more).cpu()

    def check(self, got, window=0, sinks=None, scale=None):
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        worst = 0.0
        for i, (n, l) in enumerate(self.seqs):
            rows = slice(self.start[i], self.start[i + 1])
            if n == 0:
                continue
            want, bound = attention64(self.q[rows].double(), self.kk[i].double(), self.vv[i].double(), l - n, window,
                                      sinks, scale, HALF[self.dt])
            bound = bound + (2.0 ** -24 if self.dt == F16 else 1e-30)
            err = (got[rows].double() - want).abs()
            assert not err.isnan().any(), f"sequence {i}"
            worst = max(worst, (err / bound).max().item())
        assert worst <= 1.0, f"{worst} of the bound"
        assert (got[self.start[-1]:] == 7.0).all()  # rows of no sequence


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 256, 8, 80, 96, 112, 192])
@pytest.mark.parametrize("seqs,heads,kv,page", [
    ([(1, 1)], 4, 4, 16),
    ([(1, 700)], 32, 4, 16),
    ([(1, 31), (1, 32), (1, 33), (1, 257), (1, 1)], 8, 2, 32),
    ([(5, 5), (33, 70), (1, 129), (16, 16)], 6, 2, 8),
    ([(130, 301)], 7, 1, 64),
])
def test_attention(mer, gpu, dt, d, seqs, heads, kv, page):
    b = Batch(seqs, heads, kv, d, page, dt, seed=d + heads, gap=2)
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("seqs,heads,kv,d,page", [
    ([(1, 9000), (1, 100), (1, 4097)], 8, 1, 64, 16),
    ([(1, 40000)], 16, 1, 128, 128),
    ([(300, 5000)], 4, 2, 128, 64),
    ([(700, 700)], 5, 1, 64, 16),
    ([(64, 3000), (257, 900), (1, 2500), (1, 3), (40, 40)], 16, 2, 128, 32),
    ([(20, 2600)], 12, 1, 256, 256),
])
@pytest.mark.parametrize("window,sink", [(0, False), (100, False), (1, True), (1000, True)])
def test_attention_long(mer, gpu, seqs, heads, kv, d, page, window, sink):
    b = Batch(seqs, heads, kv, d, page, BF16, seed=len(seqs) + window)
    sinks = torch.linspace(-4, 6, heads) if sink else None
    b.check(b.run(mer, gpu, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("keys", [4096, 4219, 4300, 6200, 33000])
@pytest.mark.parametrize("heads,d", [(3, 128), (16, 64), (9, 256)])
def test_attention_many_pieces(mer, gpu, keys, heads, d):
    """One unit over as many workgroups as there are stretches of 128 keys: 32,
    33, 34, 49 and all of them; three calls, whose workgroups end in other orders."""
    b = Batch([(1, keys)], heads, 1, d, 64, F16, seed=keys)
    got = [b.run(mer, gpu) for _ in range(3)]
    b.check(got[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("n,window", [(1, 33), (3, 33), (40, 33), (260, 33), (200, 0)])
def test_attention_small_weights_count(mer, gpu, n, window):
    """One key far ahead of 32 others in every window, with values of zero: what
    the others add, 2^-15 to 2^-18 of it each, is all there is."""
    seqs, heads, d = [(n, 300)], 4, 64
    b = Batch(seqs, heads, 1, d, 16, F16, seed=17)
    big = torch.arange(300) % 33 == 0
    b.q[:] = 0
    b.q[..., 0] = 1
    b.kk[0][:] = 0
    b.kk[0][:, 0, 0] = torch.where(big, 12.0, torch.linspace(-0.45, 1.6, 300)).to(F16)
    b.vv[0][:] = b.vv[0].abs() + 0.5
    b.vv[0][big] = 0
    for j in range(300):
        b.k[b.table[0, j // 16], :, j % 16] = b.kk[0][j]
        b.v[b.table[0, j // 16], :, j % 16] = b.vv[0][j]
    got = b.run(mer, gpu, scale=1.0, window=window)
    want, bound = attention64(b.q.double(), b.kk[0].double(), b.vv[0].double(), 300 - n, window, None, 1.0, HALF[F16])
    # f16 weights and outputs; an output below 2^-14 rounds by 2^-25
    assert ((got.double() - want).abs() <= bound + 2.0 ** -25).all()
    assert (want > 2.0 ** -14).all()


@pytest.mark.parametrize("n_seqs,new,keys,heads,kv,d,window", [
    (1, 5, 4000, 16, 4, 128, 0), (3, 7, 900, 9, 3, 64, 50), (3, 20, 700, 4, 4, 256, 0),  # tiles of 16
    (2, 9, 17000, 24, 8, 128, 0), (2, 8, 17500, 32, 8, 64, 900),                         # of 32
    (130, 8, 150, 8, 2, 64, 0), (70, 6, 333, 16, 4, 128, 100), (260, 17, 40, 1, 1, 256, 0),  # of 128
])
def test_attention_few_tokens(mer, gpu, n_seqs, new, keys, heads, kv, d, window):
    """A few tokens of each sequence: 17 to 32 rows of a kv head."""
    seqs = [(new - i % 2, keys - 3 * i % 37) for i in range(n_seqs)]
    b = Batch(seqs, heads, kv, d, 16, BF16, seed=n_seqs + new)
    sinks = torch.linspace(-3, 3, heads) if window else None
    b.check(b.run(mer, gpu, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("n,heads,kv,d", [(600, 4, 2, 64), (300, 20, 4, 128), (257, 2, 1, 256), (2100, 2, 1, 64)])
@pytest.mark.parametrize("more", [0, 1])
def test_attention_many_sequences(mer, gpu, n, heads, kv, d, more):
    """More sequences than a wave views at once, some without rows or keys, and
    enough of them for the workgroups of one wave."""
    seqs = [((i % 7 != 3) * (1 + more * (i % 2)), (37 * i) % 211) for i in range(n)]
    b = Batch(seqs, heads, kv, d, 8, F16, seed=n)
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("hints", [dict(max_q_len=1, max_kv_len=1), dict(max_q_len=10 ** 6, max_kv_len=10 ** 6),
                                   dict(max_q_len=3, max_kv_len=300), {}])
def test_attention_hints_do_not_matter(mer, gpu, hints):
    b = Batch([(1, 1500), (37, 400), (3, 2000), (200, 1100)], 8, 2, 64, 16, F16, seed=5)
    b.check(b.run(mer, gpu, hints=False, **hints))


def test_attention_rows_that_see_nothing(mer, gpu):
    """Sequences without keys, with fewer keys than new tokens, without rows."""
    b = Batch([(3, 0), (20, 7), (0, 50), (0, 0), (1, 0), (2, 2)], 4, 2, 64, 8, F16, seed=6, gap=3)
    for sinks in (None, torch.tensor([0.0, -50.0, 50.0, 1.0])):
        got = b.run(mer, gpu, sinks=sinks)
        b.check(got, sinks=sinks)
        assert (got[:3] == 0).all() and (got[3:3 + 13] == 0).all()


def test_attention_scores_far_apart(mer, gpu):
    """Scores of hundreds either way: the running maximum jumps from tile to tile."""
    for scale in (3.0, -3.0):
        b = Batch([(1, 3000), (40, 999)], 4, 1, 64, 16, F16, seed=7, kscale=4.0)
        b.check(b.run(mer, gpu, scale=scale), scale=scale)


def test_attention_pages_before_the_window_are_not_read(mer, gpu):
    b = Batch([(1, 1000), (30, 800)], 8, 2, 128, 16, BF16, seed=8)
    for i, (n, l) in enumerate(b.seqs):
        b.table[i, :(l - n - 99) // 16] = -1 if i else 10 ** 6
    mer.take_device_status()
    b.check(b.run(mer, gpu, window=100), window=100)
    mer.take_device_status()


@pytest.mark.parametrize("seqs,heads,kv,d", [([(1, 5000), (1, 3)], 8, 1, 128), ([(150, 900), (7, 7)], 8, 2, 64),
                                             ([(40, 6000)], 8, 1, 256)])
def test_attention_in_place(mer, gpu, seqs, heads, kv, d):
    b = Batch(seqs, heads, kv, d, 16, BF16, seed=14)
    q = b.q.to(gpu)
    cache = mer.PagedKvCache.wrap(b.k.to(gpu), b.v.to(gpu))
    args = (b.table.to(gpu), torch.tensor(b.start, dtype=torch.int32, device=gpu),
            torch.tensor([l for _, l in seqs], dtype=torch.int32, device=gpu))
    want = mer.paged_attention(cache, q, *args)
    assert mer.paged_attention(cache, q, *args, out=q) is q
    assert torch.equal(q, want)
    b.check(q.cpu())


@pytest.mark.parametrize("heads,kv,d,seqs,window,split", [
    (16, 2, 128, [(2, 75), (1, 40)], 0, False),     # 16-row tiles
    (16, 2, 64, [(4, 300), (3, 3)], 20, False),     # 32-row tiles
    (4, 1, 256, [(8, 70)], 0, False),
    (4, 2, 64, [(90, 90), (200, 333)], 0, False),   # 128-row tiles
    (8, 1, 128, [(150, 400)], 70, False),
    (2, 1, 256, [(130, 200)], 33, False),
    (8, 1, 128, [(40, 9000)], 0, True),             # their keys in chunks
])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attention_values_that_are_not_finite(mer, gpu, dt, heads, kv, d, seqs, window, split):
    """An infinity or NaN in a value reaches the rows that see its key and no
    other ones, and only its own dimension of them.  (Keys near zero, so that
    every weight is an ordinary number.)"""
    b = Batch(seqs, heads, kv, d, 16, dt, seed=12, kscale=0.1)
    marks = []  # (sequence, key, kv head, dimension, value)
    for i, (n, l) in enumerate(seqs):
        for j, x in enumerate((math.nan, math.inf, -math.inf, math.inf, -math.inf, math.nan)):
            marks.append((i, max(l - 1 - j * max(n // 4, 1), 0), j % kv, (5 * j + 3) % d if j < 4 else 8, x))
        marks.append((i, 0, 0, 11, math.inf))
    clean = [v.clone() for v in b.vv]
    for i, key, g, at, x in marks:
        b.vv[i][key, g, at] = x
        clean[i][key, g, at] = 0
        b.v[b.table[i, key // 16], g, key % 16, at] = x
    got = b.run(mer, gpu, window=window).double()
    group = heads // kv
    for i, (n, l) in enumerate(seqs):
        want, bound = attention64(b.q[b.start[i]:b.start[i + 1]].double(), b.kk[i].double(), clean[i].double(), l - n,
                                  window, None, d ** -0.5, HALF[dt])
        for g in range(kv):
            vv, rows = b.vv[i][:, g].double(), got[b.start[i]:b.start[i + 1], g * group:(g + 1) * group]
            for r in range(n):
                lo, hi = max(l - n + r + 1 - window, 0) if window else 0, l - n + r + 1
                odd = torch.where(vv[lo:hi].isfinite(), 0.0, vv[lo:hi]).sum(0)  # [d]
                for hd in range(group):
                    x, w, h = rows[r, hd], want[r, g * group + hd], bound[r, g * group + hd]
                    ok = torch.where(odd.isnan(), x.isnan(), torch.where(odd != 0, x == odd, (x - w).abs() <= h + 2.0 ** -24))
                    assert ok.all(), (i, g, r, hd, x[~ok], w[~ok], odd[~ok])


@pytest.mark.parametrize("n,l,heads,kv,d", [
    (1, 700, 8, 2, 128), (1, 6000, 8, 1, 64), (1, 40000, 4, 1, 128), (1, 3000, 3, 1, 256),  # 16-row tiles, pieces
    (3, 2000, 16, 2, 192), (6, 3000, 20, 4, 64),
    (60, 300, 4, 2, 64), (300, 900, 4, 1, 128), (40, 9000, 8, 1, 128), (130, 1000, 2, 1, 256), (70, 400, 4, 2, 80),
])
@pytest.mark.parametrize("window,sink", [(0, None), (0, 2000.0), (150, None)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attention_infinite_values_of_no_weight(mer, gpu, dt, n, l, heads, kv, d, window, sink):
    """Scores that grow with the key, so that weights far back round to zero: an
    infinity or NaN there reaches every row that sees its key all the same, in
    whatever tile, piece or chunk it lies and whatever the call is told to expect."""
    b = Batch([(n, l)], heads, kv, d, 16, dt, seed=19)
    b.q[:] = 0
    b.q[..., 0] = 1
    b.kk[0][:] = 0
    b.kk[0][..., 0] = (torch.arange(l) * (600.0 / l)).to(dt)[:, None]
    clean = b.vv[0].clone()
    for i, key in enumerate((0, 40, l // 3, l // 2, l - n - 70, l - n, l - n // 2 - 1, l - 1)):
        for j, x in enumerate((math.inf, -math.inf, math.nan)):
            at = (7 * i + 2 * j) % d
            b.vv[0][max(key, 0), i % kv, at] = x
    b.vv[0][41, 0, 7 % d] = -math.inf
    clean[~b.vv[0].isfinite()] = 0
    for j in range(l):
        b.k[b.table[0, j // 16], :, j % 16] = b.kk[0][j]
        b.v[b.table[0, j // 16], :, j % 16] = b.vv[0][j]
    sinks = None if sink is None else torch.full((heads,), sink)
    want, bound = attention64(b.q.double(), b.kk[0].double(), clean.double(), l - n, window, sinks, 1.0, HALF[dt])
    bound = bound + (2.0 ** -24 if dt == F16 else 1e-30)
    odd = torch.where(b.vv[0].isfinite(), 0.0, b.vv[0].double())  # [l, kv, d]
    rows = [odd[max(l - n + r + 1 - window, 0) if window else 0:l - n + r + 1].sum(0) for r in range(n)]
    odd = torch.stack(rows).repeat_interleave(heads // kv, 1)
    for hints in (dict(max_q_len=n, max_kv_len=l), {}, dict(max_q_len=1, max_kv_len=1), dict(max_q_len=10 ** 6)):
        got = b.run(mer, gpu, hints=False, scale=1.0, window=window, sinks=sinks, **hints).double()
        ok = torch.where(odd.isnan(), got.isnan(), torch.where(odd != 0, got == odd, (got - want).abs() <= bound))
        assert ok.all(), (hints, (~ok).nonzero()[:4], got[~ok][:4], want[~ok][:4], odd[~ok][:4])


@pytest.mark.parametrize("n,l,heads,kv,d", [(3, 75, 8, 2, 128), (6, 300, 8, 2, 64), (150, 400, 4, 2, 64), (40, 9000, 8, 1, 128)])
@pytest.mark.parametrize("x", [math.nan, math.inf])
def test_attention_key_that_is_not_finite(mer, gpu, n, l, heads, kv, d, x):
    """The last token's key: its own rows of that kv head have no answer, all
    others are as if it were not there."""
    b = Batch([(n, l)], heads, kv, d, 16, F16, seed=15)
    b.k[b.table[0, (l - 1) // 16], 0, (l - 1) % 16, 5] = x
    b.q[-1].abs_()  # its score is +inf, or NaN
    got = b.run(mer, gpu)
    group = heads // kv
    assert got[-1, :group].isnan().all()
    want, bound = attention64(b.q.double(), b.kk[0].double(), b.vv[0].double(), l - n, 0, None, d ** -0.5, HALF[F16])
    err, bound = (got.double() - want).abs(), bound + 2.0 ** -24
    assert (err[:-1] <= bound[:-1]).all() and (err[-1, group:] <= bound[-1, group:]).all()


@pytest.mark.parametrize("n,l,heads,kv", [(1, 200, 8, 2), (5, 260, 12, 2), (140, 333, 4, 2), (40, 9000, 8, 1)])
@pytest.mark.parametrize("d", [8, 64, 72, 80, 96, 112, 128, 192, 200, 256])
@pytest.mark.parametrize("x", [math.inf, -math.inf])
def test_attention_key_that_no_row_minds(mer, gpu, n, l, heads, kv, d, x):
    """Infinities in keys, against a q of the other sign: scores of -inf, so
    these keys weigh nothing and every row has the answer of the others."""
    b = Batch([(n, l)], heads, kv, d, 16, F16, seed=18)
    dims = (3, d - 1)
    for at in dims:
        b.q[..., at] = -math.copysign(1.0, x) * (b.q[..., at].abs() + 0.5)
    for key in (0, 37, l // 2, l - n - 1, max(l - n // 2 - 1, 1)):
        at = dims[key % 2]
        b.k[b.table[0, key // 16], :, key % 16, at] = x
        b.kk[0][key, :, at] = math.copysign(3e4, x)  # of q's >= 0.5: exp(-900) at most
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("n", [2, 60])
def test_attention_lengths_past_the_arrays(mer, gpu, n):
    """kv_len is cut to what the table holds, rows to those of q; negative
    lengths and starts are empty."""
    b = Batch([(n, 96)], 4, 2, 64, 16, F16, seed=16)
    cache = mer.PagedKvCache.wrap(b.k.to(gpu), b.v.to(gpu))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    table = b.table[:, :6].contiguous().to(gpu)
    got = mer.paged_attention(cache, b.q.to(gpu), table, i32(0, 2 ** 31 - 1), i32(2 ** 31 - 1))
    b.check(got.cpu())
    for start, lens in (((-5, n), (96,)), ((0, n), (96,))):
        b.check(mer.paged_attention(cache, b.q.to(gpu), table, i32(*start), i32(*lens)).cpu())
    for start, lens in (((0, n), (-1,)), ((n, 0), (96,)), ((0, -7), (96,)), ((n + 3, n + 9), (96,))):
        got = mer.paged_attention(cache, b.q.to(gpu), table, i32(*start), i32(*lens))
        assert (got == 0).all(), (start, lens)
    mer.take_device_status()


def test_attention_of_a_wide_table(mer, gpu):
    """A table of 2^30 keys a row and heads enough that 32 bits would not count
    their pieces."""
    b = Batch([(1, 300), (2, 77), (1, 0), (1, 1)], 64, 64, 8, 4096, F16, seed=13)
    table = torch.full((4, 1 << 18), -1, dtype=torch.int32)
    table[:, :b.table.shape[1]] = b.table
    b.table = table
    b.check(b.run(mer, gpu))


def test_attention_page_outside_the_cache(mer, gpu):
    """Reads as zeros, is recorded, and leaves other sequences alone."""
    b = Batch([(1, 100), (1, 90)], 2, 1, 64, 16, F16, seed=9)
    b.table[0, 2] = b.k.shape[0]
    b.kk[0][32:48] = 0
    b.vv[0][32:48] = 0
    mer.take_device_status()
    got = b.run(mer, gpu)
    with pytest.raises(mer.GpuExpertDispatchError):
        mer.take_device_status()
    b.check(got)


def test_attention_strided_and_other_stream(mer, gpu):
    b = Batch([(9, 200), (1, 64)], 4, 2, 64, 16, BF16, seed=10)
    wide = torch.zeros(b.n, 8, 64, dtype=BF16, device=gpu)
    wide[:, 2:6] = b.q.to(gpu)
    out = torch.full((b.n, 6, 64), 7.0, dtype=BF16, device=gpu)
    args = [b.table.to(gpu), torch.tensor(b.start, dtype=torch.int32, device=gpu),
            torch.tensor([l for _, l in b.seqs], dtype=torch.int32, device=gpu)]
    cache = mer.PagedKvCache.wrap(b.k.to(gpu), b.v.to(gpu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mer.paged_attention(cache, wide[:, 2:6], *args, out=out[:, 1:5])
    side.synchronize()
    assert (out[:, 0] == 7).all() and (out[:, 5] == 7).all()
    b.check(out[:, 1:5].cpu())


def test_attention_of_a_cache_past_4_gib(mer, gpu):
    """The last pages of a cache whose offsets do not fit 32 bits."""
    pages, kv, page, d = 20000, 8, 128, 128  # 5 GiB each of k and v
    cache = mer.PagedKvCache.wrap(torch.zeros(pages, kv, page, d, dtype=F16, device=gpu),
                                  torch.zeros(pages, kv, page, d, dtype=F16, device=gpu))
    g = torch.Generator().manual_seed(11)
    n = 300
    k, v = torch.randn(n, kv, d, generator=g).to(F16), torch.randn(n, kv, d, generator=g).to(F16)
    ids = torch.tensor([pages - 1, pages // 2 + 7, pages - 3], dtype=torch.int32)
    slots = (ids.to(torch.int64)[:, None] * page + torch.arange(page)).view(-1)[:n]
    mer.kv_append(cache, k.to(gpu), v.to(gpu), slots.to(gpu))
    q = torch.randn(2, 16, d, generator=g).to(F16)
    got = mer.paged_attention(cache, q.to(gpu), ids[None].to(gpu), torch.tensor([0, 2], dtype=torch.int32, device=gpu),
                              torch.tensor([n], dtype=torch.int32, device=gpu))
    want, bound = attention64(q.double(), k.double(), v.double(), n - 2, 0, None, d ** -0.5, HALF[F16])
    assert ((got.cpu().double() - want).abs() <= bound + 2.0 ** -24).all()
    del cache
    torch.cuda.empty_cache()
