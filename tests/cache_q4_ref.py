"""The cache held in 4 bits in plain torch on the CPU, for the tests: blocks of
32 elements, a scale d of five bits, codes n that stand for d (n - 8)."""
from __future__ import annotations

import torch

F16, F32, F64 = torch.float16, torch.float32, torch.float64
MOST_SCALE, MOST_VALUE = 7936.0, 65504.0


def five_bits(a):
    """a >= 0 in f64, rounded to five significant bits, half to even."""
    m, e = torch.frexp(a)
    return torch.round(m * 32) * 2.0 ** (e - 5).to(F64)


def quantise(x):
    """x [..., d] whose values are f32's, d a multiple of 32 -> (codes uint8
    [..., d / 2], scales f16 [..., d / 32]); nothing is said of what is not finite."""
    x = x.to(F64).unflatten(-1, (-1, 32))
    hi, lo = x.amax(-1), x.amin(-1)
    a = torch.where(hi >= -lo, hi, lo)
    d = five_bits(a.abs() / 8).to(F16).clamp(max=MOST_SCALE)
    d = torch.where(a > 0, -d, d)
    step = torch.where(d == 0, 1.0, d.to(F64))[..., None]
    n = (torch.round(x / step).clamp(-8, 7) + 8).to(torch.uint8)
    return (n[..., :16] | n[..., 16:] << 4).flatten(-2), d


def values(codes, scales):
    """f64 values of codes [..., d / 2] and scales [..., d / 32]."""
    b = codes.unflatten(-1, (-1, 16))
    n = torch.cat((b & 15, b >> 4), -1).to(F64) - 8
    return (n * scales.to(F64)[..., None]).flatten(-2)


def held(k, v):
    """(keys, values) [n, heads, d] as a cache holds them: a head whose key or
    value is not finite or too large is NaN in both."""
    out = [values(*quantise(torch.nan_to_num(x.to(F32), 0.0, 0.0, 0.0).clamp(-MOST_VALUE, MOST_VALUE))) for x in (k, v)]
    bad = sum((~(x.to(F64).abs() <= MOST_VALUE)).any(-1, keepdim=True) for x in (k, v)) > 0
    return tuple(torch.where(bad, torch.nan, x) for x in out)


def norm_rope64(x, w, positions, inv_freq, eps, interleaved):
    """x [t, heads, d] normed and rotated in 64 bits and rounded to f32."""
    y = x.to(F64)
    if w is not None:
        y = y / (y.pow(2).mean(2, keepdim=True) + eps).sqrt() * w.to(F64)
    if inv_freq is not None:
        half = inv_freq.numel()
        a = positions.to(F64)[:, None] * inv_freq.to(F64)
        c, s = a.cos()[:, None], a.sin()[:, None]
        i = torch.arange(half)
        at, to = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        u, v = y[..., at].clone(), y[..., to].clone()
        y = y.clone()
        y[..., at] = u * c - v * s
        y[..., to] = v * c + u * s
    return y.to(F32)


class Pages:
    """A cache's four tensors on the CPU: any codes, scales of NaN where nothing was written."""

    def __init__(self, pages, heads, page, d, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.page = page
        self.k_codes, self.v_codes = (torch.randint(0, 256, (pages, heads, page, d // 2), generator=g, dtype=torch.uint8)
                                      for _ in range(2))
        self.k_scales, self.v_scales = (torch.full((pages, heads, d // 32, page), torch.nan, dtype=F16) for _ in range(2))

    def put(self, slots, k, v):
        """Rows [n, heads, d] of f32 values to their slots."""
        at, place = slots // self.page, slots % self.page
        for x, codes, scales in ((k, self.k_codes, self.k_scales), (v, self.v_codes, self.v_scales)):
            c, s = quantise(x)
            codes[at, :, place] = c
            scales[at, :, :, place] = s

    def get(self, slots):
        """(keys, values) in f64."""
        at, place = slots // self.page, slots % self.page
        return tuple(values(c[at, :, place], s[at, :, :, place])
                     for c, s in ((self.k_codes, self.k_scales), (self.v_codes, self.v_scales)))

    def on(self, mer, gpu):
        return mer.PagedKvCacheQ4.wrap(self.k_codes.to(gpu), self.k_scales.to(gpu), self.v_codes.to(gpu),
                                       self.v_scales.to(gpu))
