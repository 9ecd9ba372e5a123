"""The cache held in 4 bits on the GPU: append, read back and attention, each
against its definition in 64 bits on the CPU.

Tolerances: append and kv_read have none.  The codes of an f32 x follow from
comparisons that are exact in f32 (a border d (n + 1/2) has ten bits); keys
that are normed and rotated in 64 bits differ from the reference's by some
2^-50 of their size before they are rounded to f32, which gives another code
with a chance of 2^-50 in 2^-3 an element.

Attention takes keys, values and f16 queries without a rounding (bf16 ones
within 2^-39 of their row's largest element), rounds the weights to f16, 2^7
times larger (2^-11 of each, or 2^-25 / 2^7 of the largest), and its answer
once; scores in f32 are off by (head_dim / 16 + 8) half steps of sum |q_d k_d|
scale, which moves a weight and the sum by as much, relatively.  The weights'
sum takes the rounded weights w (1 + r), so that their rounding moves the answer
o by sum w r (v - o) / z, at most max |r| sum w (|v| + |o|) / z.
"""
from __future__ import annotations

import itertools
import math
import threading

import pytest
import torch

import cache_q4_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HALF = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}


def inv_freq(rot, base=1e6):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).to(F32)


# ---- append and read -------------------------------------------------------

@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,kv,d,rot,interleaved,normed,page", [
    (1, 1, 32, 0, False, False, 8),
    (7, 2, 64, 64, False, True, 16),
    (33, 3, 96, 40, False, False, 32),
    (50, 8, 128, 128, True, True, 64),
    (130, 5, 128, 128, False, False, 8),
    (20, 4, 160, 8, True, False, 128),
    (19, 2, 192, 192, False, True, 16),
    (65, 3, 224, 112, True, True, 256),
    (300, 9, 256, 256, False, True, 32),
])
def test_append(mer, gpu, src, tokens, kv, d, rot, interleaved, normed, page):
    g = torch.Generator().manual_seed(tokens + d)
    row = (2.0 * torch.randn(tokens, 2 * kv * d + 16, generator=g)).to(src)
    k, v = row[:, :kv * d].view(tokens, kv, d), row[:, kv * d:2 * kv * d].view(tokens, kv, d)
    w = 1 + 0.2 * torch.randn(d, generator=g) if normed else None
    f = inv_freq(rot) if rot else None
    pos = torch.randint(0, 1 << 17, (tokens,), generator=g, dtype=torch.int32)
    pages = ref.Pages(-(-tokens // page) + 2, kv, page, d, seed=d)
    slots = torch.randperm(pages.k_codes.shape[0] * page, generator=g)[:tokens]
    skipped = torch.rand(tokens, generator=g) < 0.2
    given = torch.where(skipped, -1 - slots, slots)
    cache, dev = pages.on(mer, gpu), row.to(gpu)
    up = lambda t: None if t is None else t.to(gpu)
    part = lambda a: dev[:, a * kv * d:(a + 1) * kv * d].view(tokens, kv, d)
    mer.kv_append(cache, part(0), part(1), up(given), positions=up(pos) if rot else None, inv_freq=up(f), k_norm=up(w),
                  interleaved=interleaved)
    pages.put(slots[~skipped], ref.norm_rope64(k, w, pos, f, 1e-6, interleaved)[~skipped], v.to(F32)[~skipped])
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):  # places that no row went to stay as they were
        got, want = getattr(cache, name).cpu(), getattr(pages, name)
        assert torch.equal(got.view(torch.uint8), want.view(torch.uint8)) if name.endswith("codes") else torch.equal(
            torch.nan_to_num(got, 9.0), torch.nan_to_num(want, 9.0)), name
    want_k, want_v = pages.get(slots)
    for dt in (F32, F16, BF16):
        gk, gv = mer.kv_read(cache, up(given), out_dtype=dt)
        assert gk.dtype == dt and gk.shape == (tokens, kv, d)
        for got, want in ((gk, want_k), (gv, want_v)):
            assert torch.equal(got.cpu().double(), torch.where(skipped[:, None, None], 0.0, want))
    mer.take_device_status()


def special_rows(d):
    """Rows of one head that meet the ends of the format, f32; `tie` and the rows
    made of it have quotients that lie halfway between two codes."""
    g = torch.Generator().manual_seed(3)
    r = lambda s: s * torch.randn(d, generator=g)
    ramp = torch.linspace(-1, 1, d)
    tie = torch.arange(d).remainder(17).sub(8).to(F32)     # whole numbers: codes of a step of one
    rows = [torch.zeros(d), r(1e-3), r(3e-5), r(1e-6), r(2e-7), r(1e-8), r(1e-30), ramp, -ramp, tie, tie * 0.5,
            torch.where(torch.arange(d) % 2 == 0, 1.5, -1.5), torch.full((d,), -2.0), torch.full((d,), 65504.0),
            65504.0 * ramp, -60000.0 * ramp.abs(), r(1e4).clamp(-65504, 65504), 8 * tie + 4, r(1.0).abs(), -r(1.0).abs(),
            torch.where(torch.arange(d) % 32 == 31, 1.0, 0.0), torch.full((d,), 2.0 ** -25), torch.full((d,), 2.0 ** -21)]
    return torch.stack(rows)


@pytest.mark.parametrize("src", [F32, F16, BF16])
@pytest.mark.parametrize("d", [32, 128, 224])
def test_append_at_the_ends_of_the_format(mer, gpu, d, src):
    rows = special_rows(d).to(src)  # (bf16 takes 65504 to 65536, a head that does not fit)
    k, v = rows[:, None], rows.flip(0)[:, None]
    cache = mer.PagedKvCacheQ4(4, 8, 1, d)
    slots = torch.arange(len(rows))
    mer.kv_append(cache, k.to(gpu), v.to(gpu), slots.to(gpu))
    want = ref.held(k.to(F32), v.to(F32))
    for dt in (F32, F16):
        for got, w in zip(mer.kv_read(cache, slots.to(gpu), out_dtype=dt), want):
            assert torch.equal(got.cpu().double().nan_to_num(9e9), w.nan_to_num(9e9))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65536.0, -1e30])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_head_that_does_not_fit_reads_as_nan(mer, gpu, bad, where):
    n, kv, d = 6, 5, 96
    g = torch.Generator().manual_seed(4)
    k, v = torch.randn(n, kv, d, generator=g), torch.randn(n, kv, d, generator=g)
    x = k if where == "k" else v
    x[2, 3, 17], x[4, 0, 95], x[5, 4, 0] = bad, bad, bad
    cache = mer.PagedKvCacheQ4(1, 8, kv, d)
    slots = torch.arange(n)
    mer.kv_append(cache, k.to(gpu), v.to(gpu), slots.to(gpu))
    for got, w in zip(mer.kv_read(cache, slots.to(gpu), out_dtype=F32), ref.held(k, v)):
        assert w.isnan().sum() == 3 * d
        assert torch.equal(got.cpu().double().nan_to_num(9e9), w.nan_to_num(9e9))


def test_slots_past_the_cache(mer, gpu):
    cache = mer.PagedKvCacheQ4(2, 8, 2, 64)
    g = torch.Generator().manual_seed(5)
    k = torch.randn(4, 2, 64, generator=g)
    mer.kv_append(cache, k[:1].expand(16, 2, 64).contiguous().to(gpu), k[:1].expand(16, 2, 64).contiguous().to(gpu),
                  torch.arange(16, device=gpu))
    mer.take_device_status()
    before = cache.k_codes.clone()
    mer.kv_append(cache, k.to(gpu), k.to(gpu), torch.tensor([-1, 16, 1 << 40, -(1 << 60)], device=gpu))
    with pytest.raises(mer.GpuExpertDispatchError):
        mer.take_device_status()
    assert torch.equal(before, cache.k_codes)
    gk, gv = mer.kv_read(cache, torch.tensor([3, -5, 3, 1 << 62], device=gpu))
    with pytest.raises(mer.GpuExpertDispatchError):
        mer.take_device_status()
    want = ref.held(k[:1], k[:1])[0]
    zero = torch.zeros_like(want)
    for got in (gk, gv):
        assert torch.equal(got.cpu().double(), torch.cat((want, zero, want, zero)))


def test_read_into_strided_rows(mer, gpu):
    cache = mer.PagedKvCacheQ4(3, 16, 2, 64)
    k = torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(6))
    mer.kv_append(cache, k.to(gpu), -k.to(gpu), torch.arange(40, device=gpu))
    out = torch.full((40, 8, 64), 7.0, dtype=BF16, device=gpu)
    a, b = mer.kv_read(cache, torch.arange(39, -1, -1, device=gpu), k_out=out[:, 1:3], v_out=out[:, 5:7])
    assert a.data_ptr() == out[:, 1:3].data_ptr() and b.dtype == BF16
    want = ref.held(k, -k)
    assert torch.equal(out[:, 1:3].cpu().double(), want[0].flip(0)) and torch.equal(out[:, 5:7].cpu().double(), want[1].flip(0))
    assert (out[:, [0, 3, 4, 7]] == 7).all()
    empty = mer.kv_read(cache, torch.zeros(0, dtype=torch.int64, device=gpu))
    assert empty[0].shape == (0, 2, 64)


# ---- attention -------------------------------------------------------------

def attention64(q, k, v, first, window, sinks, scale, h):
    """One sequence: q [n, H, d], k and v [L, G, d] in float64; row i stands at
    first + i.  Returns (out, bound)."""
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
        lost = torch.where(seen, qq.abs().amax(1, keepdim=True) @ kk.abs().sum(1)[None] * abs(scale), 0.0) * 2.0 ** -39
        m = s.amax(1, keepdim=True) if keys else torch.full((n, 1), -math.inf, dtype=torch.float64)
        if sinks is not None:
            m = m.clamp(min=float(sinks[hd]))
        m = torch.where(m == -math.inf, 0.0, m)
        e = torch.exp(s - m)
        z = e.sum(1, keepdim=True)
        if sinks is not None:
            z = z + torch.exp(float(sinks[hd]) - m)
        z = torch.where(z > 0, z, 1.0)
        out[:, hd] = e @ vv / z
        weight = 2 * (d / 16 + 8) * HALF[F32] * size + 2 * lost + 64 * HALF[F32]
        rounded = e * HALF[F16] + torch.where(seen, 2.0 ** -32, 0.0)
        bound[:, hd] = (e * weight + rounded) @ vv.abs() / z + rounded.sum(1, keepdim=True) / z * out[:, hd].abs()
    return out, bound + h * out.abs()


class Batch:
    """Sequences [(new tokens, keys)] over scattered pages.  What the cache holds
    beyond them is any codes with scales of NaN."""

    def __init__(self, seqs, heads, kv, d, page, dt, seed, gap=0, spare=3, kscale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.page, self.dt = seqs, page, dt
        need = [-(-max(l, 0) // page) for _, l in seqs]
        width, total = max(need + [1]) + 1, sum(need) + spare
        order = torch.randperm(total, generator=g).to(torch.int32)
        self.table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        self.pages = ref.Pages(total, kv, page, d, seed)
        self.kk, self.vv, self.start, self.slots = [], [], [0], []
        at = 0
        for i, (n, l) in enumerate(seqs):
            l = max(l, 0)
            ids = order[at:at + need[i]]
            at += need[i]
            self.table[i, :need[i]] = ids
            slots = (ids.to(torch.int64)[:, None] * page + torch.arange(page)).view(-1)[:l]
            self.pages.put(slots, kscale * torch.randn(l, kv, d, generator=g), torch.randn(l, kv, d, generator=g))
            self.slots.append(slots)
            kk, vv = self.pages.get(slots)
            self.kk.append(kk)
            self.vv.append(vv)
            self.start.append(self.start[-1] + n)
        self.n = self.start[-1] + gap
        self.q = torch.randn(self.n, heads, d, generator=g).to(dt)

    def args(self, gpu):
        return [self.table.to(gpu), torch.tensor(self.start, dtype=torch.int32, device=gpu),
                torch.tensor([l for _, l in self.seqs], dtype=torch.int32, device=gpu)]

    def run(self, mer, gpu, hints=True, **kw):
        out = torch.full_like(self.q, 7.0, device=gpu)
        more = dict(max_q_len=max(n for n, _ in self.seqs), max_kv_len=max(l for _, l in self.seqs)) if hints else {}
        more.update(kw)
        if more.get("sinks") is not None:
            more["sinks"] = more["sinks"].to(gpu)
        return mer.paged_attention(self.pages.on(mer, gpu), self.q.to(gpu), *self.args(gpu), out=out, **more).cpu()

    def check(self, got, window=0, sinks=None, scale=None):
        scale = self.q.shape[2] ** -0.5 if scale is None else scale
        worst = 0.0
        for i, (n, l) in enumerate(self.seqs):
            rows = slice(self.start[i], self.start[i + 1])
            if n == 0:
                continue
            want, bound = attention64(self.q[rows].double(), self.kk[i], self.vv[i], l - n, window, sinks, scale,
                                      HALF[self.dt])
            bound = bound + (2.0 ** -24 if self.dt == F16 else 1e-30)
            err = (got[rows].double() - want).abs()
            assert not err.isnan().any(), f"sequence {i}"
            worst = max(worst, (err / bound).max().item())
        assert worst <= 1.0, f"{worst} of the bound"
        assert (got[self.start[-1]:] == 7.0).all()  # rows of no sequence


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("seqs,heads,kv,page", [
    ([(1, 1)], 4, 4, 16),
    ([(1, 700)], 32, 4, 16),
    ([(1, 31), (1, 32), (1, 33), (1, 64), (1, 65), (1, 257), (1, 1)], 8, 2, 32),
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
    ([(5, 2600), (5, 3100), (4, 900)], 10, 2, 96, 8),
    ([(20, 2600)], 12, 1, 256, 256),
])
@pytest.mark.parametrize("window,sink", [(0, False), (100, False), (1, True), (1000, True)])
def test_attention_long(mer, gpu, seqs, heads, kv, d, page, window, sink):
    b = Batch(seqs, heads, kv, d, page, BF16 if d != 96 else F16, seed=len(seqs) + window)
    sinks = torch.linspace(-4, 6, heads) if sink else None
    b.check(b.run(mer, gpu, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("seqs", [[(1, 700), (3, 90)], [(70, 500), (1, 40)]])
def test_hints_do_not_matter(mer, gpu, seqs):
    """Unknown lengths, and lengths that are not true."""
    b = Batch(seqs, 8, 2, 128, 16, F16, seed=21)
    b.check(b.run(mer, gpu, hints=False))
    b.check(b.run(mer, gpu, max_q_len=1, max_kv_len=1))
    b.check(b.run(mer, gpu, max_q_len=1, max_kv_len=100000))


@pytest.mark.parametrize("scale", [0.5, -0.02, 1e-6])
@pytest.mark.parametrize("n", [1, 90])
def test_scale(mer, gpu, scale, n):
    b = Batch([(n, 300)], 4, 1, 64, 16, BF16, seed=22)
    b.check(b.run(mer, gpu, scale=scale), scale=scale)


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("size", [2.0 ** -120, 2.0 ** -40, 2.0 ** 20, 2.0 ** 100])
def test_bf16_queries_beyond_f16(mer, gpu, n, size):
    """Queries whose size f16 does not have, beside a scale that makes up for it."""
    b = Batch([(n, 300)], 4, 2, 96, 16, BF16, seed=23)
    b.q = (b.q.double() * size).to(BF16)
    scale = 0.1 / size
    b.check(b.run(mer, gpu, scale=scale), scale=scale)


@pytest.mark.parametrize("keys", [4096, 4219, 4300, 6200, 33000])
@pytest.mark.parametrize("heads,d", [(3, 128), (16, 64), (9, 256)])
def test_attention_many_pieces(mer, gpu, keys, heads, d):
    """One unit over many workgroups; three calls, whose workgroups end in other orders."""
    b = Batch([(1, keys)], heads, 1, d, 64, F16, seed=keys)
    got = [b.run(mer, gpu) for _ in range(3)]
    b.check(got[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("n,window", [(1, 33), (3, 33), (40, 33), (260, 33), (200, 0)])
def test_small_weights_count(mer, gpu, n, window):
    """One key far ahead of 32 others in every window, with values of zero: what
    the others add, 2^-15 to 2^-18 of it each, is all there is."""
    seqs, heads, d = [(n, 300)], 4, 64
    b = Batch(seqs, heads, 1, d, 16, F16, seed=17)
    big = torch.arange(300) % 33 == 0
    b.q[:] = 0
    b.q[..., 0] = 1
    k, v = torch.zeros(300, 1, d), torch.randn(300, 1, d, generator=torch.Generator().manual_seed(1))
    k[big, 0, 0] = 8 * (11.0 + 0.5 * torch.arange(big.sum()) % 2)
    v[big] = 0
    b.pages.put(b.slots[0], k, v)
    b.kk[0], b.vv[0] = b.pages.get(b.slots[0])
    b.check(b.run(mer, gpu, window=window), window)


@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("d", [64, 128, 224])
def test_rows_that_see_nothing_give_zeros(mer, gpu, n, d):
    """More rows than keys, and sequences without keys or without rows."""
    b = Batch([(n, max(0, n - 2)), (1, 0), (0, 40), (2, 90)], 4, 2, d, 16, F16, seed=24)
    got = b.run(mer, gpu)
    b.check(got)
    assert (got[n:n + 1] == 0).all()
    if n > 2:
        assert (got[:2] == 0).all()


@pytest.mark.parametrize("n,keys,group", [(1, 300, 1), (6, 300, 4), (100, 400, 2), (300, 300, 4)])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("where", ["k", "v"])
def test_nan_reaches_only_the_rows_that_see_it(mer, gpu, n, keys, group, d, where):
    """Rows appended with something not finite: the rows that see the key have
    no answer, the others that of a cache without it."""
    window = 40
    b = Batch([(n, keys)], 2 * group, 2, d, 16, F16, seed=25)
    want = b.run(mer, gpu, window=window)
    cache = b.pages.on(mer, gpu)
    at = sorted({keys - n + n // 2, keys - 1, max(0, keys - n - 60)})
    k, v = (torch.randn(len(at), 2, d, generator=torch.Generator().manual_seed(d)).to(F16) for _ in range(2))
    (k if where == "k" else v)[:, 1, d - 1] = torch.tensor([math.nan, math.inf, -math.inf])[:len(at)]
    for x, t in ((k, b.kk), (v, b.vv)):  # head 0 as it was
        x[:, 0] = t[0][at, 0].to(F16)
    mer.kv_append(cache, k.to(gpu), v.to(gpu), b.slots[0][at].to(gpu))
    got = mer.paged_attention(cache, b.q.to(gpu), *b.args(gpu), window=window, max_q_len=n).cpu()
    p = keys - n + torch.arange(n)[:, None]
    sees = torch.stack([(j <= p[:, 0]) & (j > p[:, 0] - window) for j in at]).any(0)
    assert torch.equal(got[:, :group].view(torch.int16), want[:, :group].view(torch.int16))
    assert got[sees][:, group:].isnan().all()
    assert torch.equal(got[~sees][:, group:].view(torch.int16), want[~sees][:, group:].view(torch.int16))


@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("d", [64, 128, 192])
def test_scales_of_values_that_are_not_finite_count_as_zero(mer, gpu, n, d):
    """In a cache that other code wrote; 8192 and more likewise."""
    b = Batch([(n, 200)], 3, 1, d, 16, F16, seed=26)
    for j, wild in ((3, math.nan), (77, math.inf), (130, -math.inf), (199, 8192.0), (64, -65504.0)):
        s = int(b.slots[0][j])
        b.pages.v_scales[s // 16, 0, j % (d // 32), s % 16] = wild
        b.vv[0][j, 0, j % (d // 32) * 32:][:32] = 0
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("seqs", [[(1, 300), (2, 80)], [(5, 300)], [(100, 400), (1, 90)]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_queries_that_are_not_finite(mer, gpu, dt, seqs, d):
    """Their own rows have no answer, the others the one that they have without them."""
    b = Batch(seqs, 8, 2, d, 16, dt, seed=41)
    want = b.run(mer, gpu)
    bad = {(0, 3): math.nan, (b.n - 1, 0): math.inf, (b.n // 2, 7): -math.inf}
    for (row, head), x in bad.items():
        b.q[row, head, d - 1] = x
    got = b.run(mer, gpu)
    for row, head in bad:
        assert got[row, head].isnan().all()
        got[row, head] = want[row, head]
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("n", [1, 50])
def test_page_outside_the_cache(mer, gpu, page, n):
    """Reads as zeros, is recorded, and leaves other sequences alone."""
    b = Batch([(n, 200), (1, 90)], 2, 1, 64, page, F16, seed=9)
    b.table[0, 1] = b.pages.k_codes.shape[0]
    b.table[0, 64 // page + 1] = -7
    b.kk[0][page:2 * page] = b.vv[0][page:2 * page] = 0
    b.kk[0][64 + page:][:page] = b.vv[0][64 + page:][:page] = 0
    mer.take_device_status()
    got = b.run(mer, gpu)
    with pytest.raises(mer.GpuExpertDispatchError):
        mer.take_device_status()
    b.check(got)


def test_pages_that_no_row_sees_are_not_looked_up(mer, gpu):
    """Beyond kv_len and before every row's window the table may hold anything."""
    for n, l, window in ((1, 300, 50), (2, 131, 64), (90, 400, 33)):
        b = Batch([(n, l)], 4, 2, 128, 16, F16, seed=27)
        first = max(0, l - n - window + 1)
        b.table[0, :first // 16] = 1 << 30
        b.table[0, -(-l // 16):] = -(1 << 31)
        mer.take_device_status()
        b.check(b.run(mer, gpu, window=window), window)
        mer.take_device_status()


@pytest.mark.parametrize("dt", [F16, BF16])
def test_in_place_and_strided(mer, gpu, dt):
    b = Batch([(9, 200), (1, 64), (70, 70)], 4, 2, 64, 16, dt, seed=10)
    cache, args = b.pages.on(mer, gpu), b.args(gpu)
    want = mer.paged_attention(cache, b.q.to(gpu), *args)
    b.check(want.cpu())
    q = b.q.to(gpu)
    assert mer.paged_attention(cache, q, *args, out=q) is q and torch.equal(q, want)
    wide = torch.zeros(b.n, 8, 64, dtype=dt, device=gpu)
    wide[:, 2:6] = b.q.to(gpu)
    out = torch.full((b.n, 6, 64), 7.0, dtype=dt, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mer.paged_attention(cache, wide[:, 2:6], *args, out=out[:, 1:5])
    side.synchronize()
    assert torch.equal(out[:, 1:5], want) and (out[:, 0] == 7).all() and (out[:, 5] == 7).all()
    mer.stream_release(side)


def test_spans_outside_the_arrays(mer, gpu):
    """Starts and lengths that the arrays do not hold are cut to them."""
    b = Batch([(2, 90), (3, 40)], 4, 2, 64, 16, F16, seed=28)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    cache, q, table = b.pages.on(mer, gpu), b.q.to(gpu), b.table.to(gpu)
    for start, lens in (((0, 2, 2 ** 31 - 1), (90, 40)), ((-5, 2, 5), (90, 40)), ((0, 2, 1), (90, 40))):
        got = mer.paged_attention(cache, q, table, i32(*start), i32(*lens)).cpu()
        assert got.isfinite().all()
        if start[-1] > 2:
            b.check(got)
    mer.take_device_status()
    mer.paged_attention(cache, q, table, i32(0, 2, 5), i32(-3, 2 ** 31 - 1))
    with pytest.raises(mer.GpuExpertDispatchError):  # the table's unused places
        mer.take_device_status()
    z = lambda n: torch.zeros(n, 4, 64, dtype=F16, device=gpu)
    assert mer.paged_attention(cache, z(0), table, i32(0, 0, 0), i32(5, 5)).shape == (0, 4, 64)
    assert (mer.paged_attention(cache, z(3), table[:, :0], i32(0, 1, 3), i32(5, 5)) == 0).all()


def test_many_sequences(mer, gpu):
    """More than the walk over the sequences has in view, short and empty ones among them."""
    g = torch.Generator().manual_seed(29)
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    b = Batch([(int(l > 0), l) for l in lens], 4, 2, 64, 16, F16, seed=29)
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("d,page", [(64, 16), (96, 8), (128, 64), (256, 32)])
@pytest.mark.parametrize("window,sink", [(0, False), (90, True)])
def test_many_units(mer, gpu, d, page, window, sink):
    """Single tokens and a short draft of as many units as give every wave a
    workgroup of its own, one of them cut into many pieces."""
    g = torch.Generator().manual_seed(35)
    lens = torch.randint(0, 500, (60,), generator=g).tolist() + [9000, 1, 128, 129]
    b = Batch([(1 + i % 2, max(l, 1 + i % 2)) for i, l in enumerate(lens)], 8, 4, d, page, BF16 if d == 128 else F16, seed=d, gap=1)
    sinks = torch.linspace(-3, 3, 8) if sink else None
    b.check(b.run(mer, gpu, window=window, sinks=sinks), window, sinks)


@pytest.mark.parametrize("n,heads,kv", [(1, 16, 16), (5, 64, 16), (1, 5, 5)])
@pytest.mark.parametrize("seqs", [70, 250])
def test_more_units_than_workgroups(mer, gpu, n, heads, kv, seqs):
    g = torch.Generator().manual_seed(39)
    lens = torch.randint(n, 400, (seqs,), generator=g).tolist()
    b = Batch([(n, l) for l in lens], heads, kv, 32, 16, BF16, seed=40)
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128, 224])
@pytest.mark.parametrize("window", [0, 70])
def test_drafts(mer, gpu, dt, d, window):
    """17 to 32 rows of a kv head, over caches of most lengths at once."""
    b = Batch([(8, 900), (5, 2000), (6, 37), (8, 8), (7, 0), (0, 50), (8, 4100), (1, 1), (3, 128)], 8, 2, d, 16, dt, seed=36, gap=3)
    b.check(b.run(mer, gpu, window=window), window)


@pytest.mark.parametrize("keys", [1000, 1024, 1025, 4000, 4224, 5000, 5121, 30000])
@pytest.mark.parametrize("seqs", [1, 3])
def test_workgroups_that_begin_with_a_unit(mer, gpu, keys, seqs):
    """Lengths on both sides of where a stretch a quarter longer gives every unit
    workgroups of its own, equal and ragged."""
    b = Batch([(1, keys - 700 * i) for i in range(seqs)], 16, 4, 64, 128, F16, seed=keys)
    b.check(b.run(mer, gpu))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_unknown_pages_of_eight_keys_in_large_tiles(mer, gpu, d):
    """A share of a tile of a prompt holds two such pages, each known or not."""
    page = 8
    b = Batch([(50, 200), (70, 90)], 4, 1, d, page, BF16, seed=37)
    for at in (0, 3, 4, 5, 10, 24):
        b.table[0, at] = b.pages.k_codes.shape[0] + at
        b.kk[0][at * page:(at + 1) * page] = b.vv[0][at * page:(at + 1) * page] = 0
    mer.take_device_status()
    got = b.run(mer, gpu)
    with pytest.raises(mer.GpuExpertDispatchError):
        mer.take_device_status()
    b.check(got)


def test_a_table_of_2_to_30_keys_a_row(mer, gpu):
    """More granules than the small tiles count in 32 bits: the 128-row tiles take the call."""
    seqs = [(1, 100), (1, 3), (0, 0), (2, 700)]
    b = Batch(seqs, 64, 64, 32, 256, F16, seed=38)
    table = torch.full((4, (1 << 30) // 256), -1, dtype=torch.int32, device=gpu)
    table[:, :b.table.shape[1]] = b.table.to(gpu)
    out = torch.full_like(b.q, 7.0, device=gpu)
    mer.take_device_status()
    mer.paged_attention(b.pages.on(mer, gpu), b.q.to(gpu), table, *b.args(gpu)[1:], max_q_len=2, max_kv_len=700, out=out)
    mer.take_device_status()
    b.check(out.cpu())


def test_a_cache_past_4_gib(mer, gpu):
    """The last pages of a cache whose offsets do not fit 32 bits."""
    pages, kv, page, d = 40000, 8, 256, 128  # 4.9 GiB of codes of k and of v
    z = lambda *s, dtype: torch.zeros(*s, dtype=dtype, device=gpu)
    cache = mer.PagedKvCacheQ4.wrap(*(z(pages, kv, page, d // 2, dtype=torch.uint8) if i % 2 == 0 else
                                      z(pages, kv, d // 32, page, dtype=F16) for i in range(4)))
    g = torch.Generator().manual_seed(11)
    n = 600
    k, v = torch.randn(n, kv, d, generator=g), torch.randn(n, kv, d, generator=g)
    ids = torch.tensor([pages - 1, pages // 2 + 7, pages - 3], dtype=torch.int32)
    slots = (ids.to(torch.int64)[:, None] * page + torch.arange(page)).view(-1)[:n]
    mer.kv_append(cache, k.to(gpu), v.to(gpu), slots.to(gpu))
    kk, vv = ref.held(k, v)
    for got, want in zip(mer.kv_read(cache, slots.to(gpu), out_dtype=F32), (kk, vv)):
        assert torch.equal(got.cpu().double(), want)
    for rows in (2, 40):
        q = torch.randn(rows, 16, d, generator=g).to(F16)
        got = mer.paged_attention(cache, q.to(gpu), ids[None].to(gpu), torch.tensor([0, rows], dtype=torch.int32, device=gpu),
                                  torch.tensor([n], dtype=torch.int32, device=gpu))
        want, bound = attention64(q.double(), kk, vv, n - rows, 0, None, d ** -0.5, HALF[F16])
        assert ((got.cpu().double() - want).abs() <= bound + 2.0 ** -24).all()
    del cache
    torch.cuda.empty_cache()


# ---- the operators together ------------------------------------------------

class Steps:
    """Steps of a layer's attention side over a cache held in 4 bits: norms and
    rotation of the queries, append, attention, and the keys read back."""

    def __init__(self, mer, gpu, counts, heads, kv, d, page, width, seed):
        g = torch.Generator().manual_seed(seed)
        self.mer, self.counts, self.shape, self.page, self.g = mer, counts, (heads, kv, d), page, g
        self.n, seqs = sum(counts), len(counts)
        self.cache = mer.PagedKvCacheQ4(seqs * width, page, kv, d, device=gpu)
        self.table = torch.randperm(seqs * width, generator=g).to(torch.int32).view(seqs, width)
        zeros = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=gpu)
        for t in (self.cache.k_scales, self.cache.v_scales):
            t.zero_()
        self.row = zeros(self.n, (heads + 2 * kv) * d, dtype=BF16)
        self.slots, self.pos = zeros(self.n, dtype=torch.int64), zeros(self.n, dtype=torch.int32)
        self.start = torch.tensor([0] + list(itertools.accumulate(counts)), dtype=torch.int32, device=gpu)
        self.lens, self.dev_table = zeros(seqs, dtype=torch.int32), self.table.to(gpu)
        self.q16, self.out = zeros(self.n, heads, d, dtype=BF16), zeros(self.n, heads, d, dtype=BF16)
        self.back = [zeros(self.n, kv, d) for _ in range(2)]
        self.freq, self.kn = inv_freq(d).to(gpu), (1 + 0.1 * torch.randn(d, generator=g)).to(gpu)
        self.width = width

    def load(self, lens):
        """New inputs: sequences of these lengths, the new tokens included."""
        slots, pos = [], []
        for i, (c, l) in enumerate(zip(self.counts, lens)):
            for at in range(l - c, l):
                pos.append(at)
                slots.append(int(self.table[i, at // self.page]) * self.page + at % self.page)
        self.slots.copy_(torch.tensor(slots))
        self.pos.copy_(torch.tensor(pos, dtype=torch.int32))
        self.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.row.copy_(torch.randn(self.row.shape, generator=self.g))

    def run(self, out):
        heads, kv, d = self.shape
        row, n, mer = self.row, self.n, self.mer
        k, v = (row[:, (heads + i * kv) * d:(heads + (i + 1) * kv) * d].view(n, kv, d) for i in (0, 1))
        mer.qk_norm_rope(row[:, :heads * d].view(n, heads, d), None, self.pos, self.freq, q_out=self.q16)
        mer.kv_append(self.cache, k, v, self.slots, positions=self.pos, inv_freq=self.freq, k_norm=self.kn)
        mer.paged_attention(self.cache, self.q16, self.dev_table, self.start, self.lens, out=out,
                            max_q_len=max(self.counts), max_kv_len=self.width * self.page)
        mer.kv_read(self.cache, self.slots, k_out=self.back[0], v_out=self.back[1])


def test_a_prompt_and_its_decode_steps(mer, gpu):
    """A prompt in chunks, then single tokens: every step against the formula
    over all that was appended."""
    heads, kv, d, page, total = 8, 2, 128, 16, 150
    g = torch.Generator().manual_seed(30)
    steps = [70, 41, 5] + [1] * 6
    ids = torch.randperm(12, generator=g).to(torch.int32)
    cache = mer.PagedKvCacheQ4(12, page, kv, d)
    f, kn = inv_freq(d), 1 + 0.1 * torch.randn(d, generator=g)
    kk, vv, at = [], [], 0
    for n in steps:
        row = torch.randn(n, (heads + 2 * kv) * d, generator=g).to(F16)
        pos = torch.arange(at, at + n, dtype=torch.int32)
        slots = ids[(pos // page).long()].to(torch.int64) * page + pos % page
        dev = row.to(gpu)
        part = lambda a, b: dev[:, a * d:b * d].view(n, b - a, d)
        q, _ = mer.qk_norm_rope(part(0, heads), None, pos.to(gpu), f.to(gpu))
        mer.kv_append(cache, part(heads, heads + kv), part(heads + kv, heads + 2 * kv), slots.to(gpu), positions=pos.to(gpu),
                      inv_freq=f.to(gpu), k_norm=kn.to(gpu))
        k = ref.norm_rope64(row[:, heads * d:(heads + kv) * d].view(n, kv, d), kn, pos, f, 1e-6, False)
        k, v = ref.held(k, row[:, (heads + kv) * d:].view(n, kv, d).to(F32))
        kk.append(k)
        vv.append(v)
        at += n
        got = mer.paged_attention(cache, q, ids[None].to(gpu), torch.tensor([0, n], dtype=torch.int32, device=gpu),
                                  torch.tensor([at], dtype=torch.int32, device=gpu), max_q_len=n, max_kv_len=total)
        want, bound = attention64(q.cpu().double(), torch.cat(kk), torch.cat(vv), at - n, 0, None, d ** -0.5, HALF[F16])
        assert ((got.cpu().double() - want).abs() <= bound + 2.0 ** -24).all(), f"step of {n} at {at}"
    slots = ids[torch.arange(at) // page].to(torch.int64) * page + torch.arange(at) % page
    for got, want in zip(mer.kv_read(cache, slots.to(gpu), out_dtype=F32), (torch.cat(kk), torch.cat(vv))):
        assert torch.equal(got.cpu().double(), want)
    mer.take_device_status()


def test_graphs_of_both_caches_on_one_stream(mer, gpu):
    """A decode step and a step with a chunk over caches in 4 bits, captured on
    one stream and replayed in turn over new inputs and growing lengths, with
    eager work and a 16-bit cache's attention between; every replay equals the
    eager call."""
    s = torch.cuda.Stream(device=gpu)
    steps = [Steps(mer, gpu, (1, 1, 1, 1), 8, 2, 128, 16, 160, 31), Steps(mer, gpu, (200, 1, 33), 8, 2, 64, 16, 160, 32)]
    other = Steps(mer, gpu, (1, 3), 4, 1, 128, 8, 40, 33)
    g = torch.Generator().manual_seed(34)
    kv16 = mer.PagedKvCache.wrap(*(torch.randn(40, 2, 16, 64, generator=g).to(BF16).to(gpu) for _ in range(2)))
    q16 = torch.randn(1, 4, 64, generator=g).to(BF16).to(gpu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    args16 = (torch.arange(40, dtype=torch.int32, device=gpu)[None], i32(0, 1), i32(600))
    graphs = []
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        first16 = mer.paged_attention(kv16, q16, *args16)
        for st in [*steps, other]:
            st.load([300] * len(st.counts))
            st.run(st.out)  # grows the workspace before capture
    s.synchronize()
    for st in steps:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            st.run(st.out)
        graphs.append(gr)
    for rep in range(4):
        for i, st in enumerate(steps):
            st.load([201 + 577 * rep + 37 * j for j in range(len(st.counts))])
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                graphs[i].replay()
                other.run(other.out)
                again16 = mer.paged_attention(kv16, q16, *args16)
            torch.cuda.synchronize()
            got, back = st.out.clone(), [t.clone() for t in st.back]
            codes = st.cache.k_codes.clone()
            want = torch.zeros_like(got)
            with torch.cuda.stream(s):
                st.run(want)
            torch.cuda.synchronize()
            assert torch.isfinite(want).all() and torch.equal(got, want), f"replay {rep} of graph {i}"
            assert torch.equal(codes, st.cache.k_codes) and all(torch.equal(a, b) for a, b in zip(back, st.back))
            assert torch.equal(first16, again16)
    mer.take_device_status()
    del graphs
    mer.stream_release(s)


def test_two_streams_at_once(mer, gpu):
    streams = [torch.cuda.Stream(device=gpu) for _ in range(2)]
    steps = [Steps(mer, gpu, (1,) * 8, 8, 2, 128, 16, 60, 41), Steps(mer, gpu, (120, 7), 8, 1, 64, 16, 60, 42)]
    want, outs = [], []
    for st in steps:
        st.load([800 + 9 * i for i in range(len(st.counts))])
        st.run(st.out)
        torch.cuda.synchronize()
        want.append(st.out.clone())
        outs.append([torch.zeros_like(st.out) for _ in range(6)])
    torch.cuda.synchronize()
    for i in range(6):
        for s, st, o in zip(streams, steps, outs):
            with torch.cuda.stream(s):
                st.run(o[i])
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)
    for s in streams:
        mer.stream_release(s)


def test_threads_with_a_stream_each(mer, gpu):
    steps = [Steps(mer, gpu, (1,) * 6, 8, 2, 128, 16, 60, 51), Steps(mer, gpu, (90, 7), 8, 1, 64, 16, 60, 52),
             Steps(mer, gpu, (5, 3, 8), 8, 2, 128, 16, 60, 53)]
    want, outs, errors = [], [], []
    for st in steps:
        st.load([700 + 9 * i for i in range(len(st.counts))])
        st.run(st.out)
        torch.cuda.synchronize()
        want.append(st.out.clone())
        outs.append([torch.zeros_like(st.out) for _ in range(8)])
    streams = [torch.cuda.Stream(device=gpu) for _ in steps]
    torch.cuda.synchronize()

    def work(s, st, out):
        try:
            with torch.cuda.stream(s):
                for o in out:
                    st.run(o)
            s.synchronize()
        except BaseException as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(streams, steps, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)
    for s in streams:
        mer.stream_release(s)


def test_smaller_calls_keep_the_workspace(mer, gpu):
    """Of this cache and of a 16-bit one on the same stream: a captured decode step
    gives its answer after all of them."""
    g = torch.Generator().manual_seed(54)
    calls = [Batch([(n, 4096)], 16, 4, 128, 64, BF16, seed=55 + n) for n in (600, 1, 300, 20, 5)]
    made = []
    for b in calls:
        made.append((b.pages.on(mer, gpu), b.q.to(gpu), *b.args(gpu), torch.zeros_like(b.q, device=gpu), b.q.shape[0]))
    kv16 = mer.PagedKvCache.wrap(*(torch.randn(64, 4, 64, 128, generator=g).to(BF16).to(gpu) for _ in range(2)))

    def run(c, out=None, cache=None):
        cache4, q, table, start, lens, mine, n = c
        mer.paged_attention(cache or cache4, q, table, start, lens, max_q_len=n, max_kv_len=4096, out=mine if out is None else out)

    table16 = torch.arange(64, dtype=torch.int32, device=gpu)[None]
    s = torch.cuda.Stream(device=gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        run(made[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        run(made[1])
    free = torch.cuda.mem_get_info(gpu)[0]
    for rep in range(3):
        with torch.cuda.stream(s):
            for c in made[1:]:
                run(c)
                run((None, c[1], table16, c[3], c[4], torch.zeros_like(c[5]), c[6]), cache=kv16)
            made[1][5].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got, want = made[1][5].clone(), torch.zeros_like(made[1][5])
        with torch.cuda.stream(s):
            run(made[1], out=want)
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {rep}"
        if rep:
            assert torch.cuda.mem_get_info(gpu)[0] == free, "a smaller call made the workspace grow"
        free = torch.cuda.mem_get_info(gpu)[0]
    calls[1].check(want.cpu())
    del graph
    mer.stream_release(s)


def test_capture_without_a_workspace_is_refused(mer, gpu):
    b = Batch([(1, 300)], 4, 2, 64, 16, F16, seed=56)
    cache, q, args = b.pages.on(mer, gpu), b.q.to(gpu), b.args(gpu)
    out = torch.zeros_like(q)
    s = torch.cuda.Stream(device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out.zero_()
        with pytest.raises(mer.GpuExpertDispatchError) as e:
            mer.paged_attention(cache, q, *args, out=out, max_q_len=1, max_kv_len=300)
    assert e.value.kind == mer.GpuExpertDispatchErrorKind.PhysicalCapacity
    with torch.cuda.stream(s):
        mer.paged_attention(cache, q, *args, out=out, max_q_len=1, max_kv_len=300)
    s.synchronize()
    b.check(out.cpu())
    del graph
    mer.stream_release(s)


def test_python_refusals(mer, gpu):
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=gpu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    cache = mer.PagedKvCacheQ4(4, 16, 2, 64)
    att = lambda **kw: mer.paged_attention(**{**dict(cache=cache, q=z(2, 4, 64), block_table=i32(0, 1, 2, 3).view(1, 4),
                                                     q_start=i32(0, 2), kv_len=i32(20)), **kw})
    app = lambda **kw: mer.kv_append(**{**dict(cache=cache, k=z(2, 2, 64), v=z(2, 2, 64),
                                               slots=torch.arange(2, device=gpu)), **kw})
    read = lambda **kw: mer.kv_read(**{**dict(cache=cache, slots=torch.arange(2, device=gpu)), **kw})
    for t in (cache.k_scales, cache.v_scales):
        t.zero_()
    att(), app(), read()
    for call, bad in [(att, dict(q=z(2, 4, 64, dtype=F32))), (att, dict(q=z(2, 4, 64, dtype=torch.float64))),
                      (att, dict(q=z(2, 4, 64, dtype=torch.int16))), (att, dict(q=z(2, 4, 128))), (att, dict(scale=0.0)),
                      (att, dict(window=-1)), (att, dict(kv_len=i32(20, 1))), (att, dict(out=z(2, 4, 64, dtype=BF16))),
                      (att, dict(q=z(2, 3, 64))), (app, dict(k=z(2, 2, 128))), (app, dict(v=z(2, 2, 64, dtype=BF16))),
                      (app, dict(slots=i32(0, 1))), (app, dict(slots=torch.arange(2))), (read, dict(slots=i32(0, 1))),
                      (read, dict(slots=torch.arange(4, device=gpu)[::2])), (read, dict(out_dtype=torch.float64)),
                      (read, dict(k_out=z(2, 2, 32))), (read, dict(k_out=z(2, 2, 64), v_out=z(2, 2, 64, dtype=F32))),
                      (read, dict(k_out=z(2, 2, 64).cpu()))]:
        with pytest.raises((ValueError, TypeError, mer.InvalidLayout, mer.GpuExpertDispatchError, mer.ExpertWeightsError)):
            call(**bad)
    torch.cuda.synchronize()
