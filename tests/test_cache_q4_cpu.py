"""The cache held in 4 bits without a GPU: refusals of the entry points
(arguments are checked before any device work), and the format's own promises."""
from __future__ import annotations

import ctypes

import pytest
import torch

import cache_q4_ref as ref

BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 255) & ~255  # an aligned address that nothing reads


@pytest.fixture
def abi(mer):
    return mer._lib


def cache(abi, **kw):
    f = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, page_size=16, n_kv_heads=2, head_dim=64, n_pages=4)
    f.update(kw)
    return ctypes.byref(abi.MerKvCacheQ4(*f.values()))


def append(abi, c=None, **kw):
    f = dict(cache=c if c is not None else cache(abi), in_type=1, n=4, k=P, ks=128, v=P, vs=128, slots=P, pos=P,
             freq=P, rot=64, interleaved=0, kn=P, eps=1e-6, stream=None)
    f.update(kw)
    return abi.lib().mer_hip_kv_append_q4(*f.values())


def read(abi, c=None, **kw):
    f = dict(cache=c if c is not None else cache(abi), out_type=1, n=4, slots=P, k=P, ks=128, v=P, vs=128, stream=None)
    f.update(kw)
    return abi.lib().mer_hip_kv_read_q4(*f.values())


def attention(abi, c=None, **kw):
    f = dict(cache=c if c is not None else cache(abi), type=1, seqs=2, n=4, h=4, q=P, qs=256, table=P, width=4, start=P,
             lens=P, mq=0, mk=0, scale=0.0, window=0, sinks=None, out=P, os=256, stream=None)
    f.update(kw)
    return abi.lib().mer_hip_paged_attention_q4(*f.values())


def test_good_arguments_get_as_far_as_the_device(abi):
    if torch.cuda.is_available():
        pytest.skip("would run on the GPU")
    for call in (append, read, attention):
        assert call(abi) == abi.Status.NOT_INITIALIZED
        assert call(abi, n=0) == 0  # nothing to do
    assert attention(abi, seqs=0) == 0


@pytest.mark.parametrize("change,status", [
    (dict(k_codes=0), "INVALID_LAYOUT"), (dict(v_scales=0), "INVALID_LAYOUT"), (dict(v_codes=P + 8), "MISALIGNED"),
    (dict(k_scales=P + 2), "MISALIGNED"), (dict(page_size=4), "INVALID_LAYOUT"), (dict(page_size=24), "INVALID_LAYOUT"),
    (dict(page_size=8192), "INVALID_LAYOUT"), (dict(n_kv_heads=0), "INVALID_LAYOUT"),
    (dict(n_kv_heads=2049), "INVALID_LAYOUT"), (dict(head_dim=0), "INVALID_LAYOUT"), (dict(head_dim=68), "INVALID_LAYOUT"),
    (dict(head_dim=80), "INVALID_LAYOUT"), (dict(head_dim=288), "SHAPE_EXCEEDS_WORKSPACE"), (dict(n_pages=0), "INVALID_LAYOUT"),
    (dict(n_pages=1 << 31), "INVALID_LAYOUT"),
])
def test_cache_refused(abi, change, status):
    for call in (append, read, attention):
        assert call(abi, cache(abi, **change)) == abi.Status[status]
        assert abi.last_error()[0] == abi.Status[status] and abi.last_error()[1]


def test_null_cache_refused(abi):
    for call in (append, read, attention):
        assert call(abi, cache=None) == abi.Status.INVALID_LAYOUT


@pytest.mark.parametrize("change,status", [
    (dict(in_type=3), "UNSUPPORTED_DTYPE"), (dict(k=None), "INVALID_LAYOUT"), (dict(v=P + 4), "MISALIGNED"),
    (dict(ks=132), "MISALIGNED"), (dict(vs=120), "INVALID_LAYOUT"), (dict(slots=None), "INVALID_LAYOUT"),
    (dict(pos=None), "INVALID_LAYOUT"), (dict(n=1 << 25), "SHAPE_EXCEEDS_WORKSPACE"), (dict(slots=P + 4), "MISALIGNED"),
    (dict(pos=P + 1), "MISALIGNED"), (dict(eps=-1.0), "INVALID_LAYOUT"), (dict(rot=12), "INVALID_LAYOUT"),
    (dict(rot=72), "INVALID_LAYOUT"), (dict(freq=0), "INVALID_LAYOUT"), (dict(kn=P + 4), "MISALIGNED"),
])
def test_append_refuses(abi, change, status):
    assert append(abi, **change) == abi.Status[status]


@pytest.mark.parametrize("change,status", [
    (dict(out_type=4), "UNSUPPORTED_DTYPE"), (dict(k=None), "INVALID_LAYOUT"), (dict(v=None), "INVALID_LAYOUT"),
    (dict(k=P + 8), "MISALIGNED"), (dict(ks=132), "MISALIGNED"), (dict(vs=120), "INVALID_LAYOUT"),
    (dict(slots=None), "INVALID_LAYOUT"), (dict(slots=P + 4), "MISALIGNED"), (dict(n=1 << 25), "SHAPE_EXCEEDS_WORKSPACE"),
])
def test_read_refuses(abi, change, status):
    assert read(abi, **change) == abi.Status[status]


@pytest.mark.parametrize("change,status", [
    (dict(type=0), "UNSUPPORTED_DTYPE"), (dict(type=2), "UNSUPPORTED_DTYPE"), (dict(h=3), "INVALID_LAYOUT"),
    (dict(h=0), "INVALID_LAYOUT"), (dict(seqs=(1 << 20) + 1), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(width=(1 << 26) + 1), "SHAPE_EXCEEDS_WORKSPACE"), (dict(q=None), "INVALID_LAYOUT"), (dict(qs=250), "MISALIGNED"),
    (dict(out=P + 6), "MISALIGNED"), (dict(table=None), "INVALID_LAYOUT"), (dict(start=P + 2), "MISALIGNED"),
    (dict(lens=P + 1), "MISALIGNED"), (dict(start=None), "INVALID_LAYOUT"), (dict(lens=None), "INVALID_LAYOUT"),
    (dict(n=1 << 25), "SHAPE_EXCEEDS_WORKSPACE"), (dict(scale=float("inf")), "INVALID_LAYOUT"),
    (dict(scale=float("nan")), "INVALID_LAYOUT"), (dict(scale=2.36e38), "INVALID_LAYOUT"), (dict(sinks=P + 2), "MISALIGNED"),
])
def test_attention_refuses(abi, change, status):
    assert attention(abi, **change) == abi.Status[status]


def tensors(pages=2, heads=1, page=8, d=64):
    codes, scales = torch.zeros(pages, heads, page, d // 2, dtype=torch.uint8), torch.zeros(pages, heads, d // 32, page).half()
    return [codes, scales, codes.clone(), scales.clone()]


@pytest.mark.parametrize("which,change,error", [
    (0, lambda t: t.to(torch.int8), TypeError), (1, lambda t: t.float(), TypeError), (3, lambda t: t.bfloat16(), TypeError),
    (0, lambda t: t[:1], ValueError), (2, lambda t: t[..., :16].contiguous(), ValueError),
    (1, lambda t: t.transpose(2, 3), ValueError), (1, lambda t: t[:, :, :1], ValueError),
    (0, lambda t: torch.cat((t, t), 3)[..., ::2], ValueError), (0, lambda t: t[0], ValueError),
    (0, lambda t: t[..., :8].contiguous(), ValueError),
])
def test_wrap_refuses(mer, which, change, error):
    t = tensors()
    mer.PagedKvCacheQ4.wrap(*t)
    t[which] = change(t[which])
    with pytest.raises(error):
        mer.PagedKvCacheQ4.wrap(*t)


def test_python_refusals(mer):
    with pytest.raises(ValueError):
        mer.PagedKvCacheQ4(2, 16, 1, 80, device="cpu")
    q4 = mer.PagedKvCacheQ4(2, 16, 1, 64, device="cpu")
    assert q4.k_codes.shape == (2, 1, 16, 32) and q4.v_scales.shape == (2, 1, 2, 16)
    with pytest.raises(ValueError):  # not on a device
        mer.kv_read(q4, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(TypeError):
        mer.kv_read(mer.PagedKvCache.wrap(*(torch.zeros(2, 1, 8, 64).half(),) * 2), torch.zeros(1, dtype=torch.int64))


def test_the_tensors_of_a_cache_cannot_be_replaced(mer):
    t = tensors()
    c = mer.PagedKvCacheQ4.wrap(*t)
    for name, x in zip(("k_codes", "k_scales", "v_codes", "v_scales"), t):
        with pytest.raises(AttributeError):
            setattr(c, name, x.clone())
        assert getattr(c, name) is x and getattr(c._desc, name) == x.data_ptr()


# ---- the format ------------------------------------------------------------

@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 3e4])
def test_values_are_exact_in_both_half_types(t, size):
    """Five bits of scale and three of n - 8 (or one, of -8) fit bf16's eight;
    f16's subnormals are its own multiples."""
    x = size * torch.randn(200, 256, generator=torch.Generator().manual_seed(1))
    y = ref.values(*ref.quantise(x))
    assert torch.equal(y.to(t).double(), y)


def test_the_error_of_a_block():
    """Half a step, or a whole one at the end that the codes lack (n - 8 = 8);
    the scale itself is off by 2^-5 of it at most."""
    x = torch.randn(500, 128, generator=torch.Generator().manual_seed(2))
    codes, d = ref.quantise(x)
    err = (ref.values(codes, d) - x.double()).abs().unflatten(-1, (-1, 32)) / d.double().abs()[..., None]
    most = x.abs().unflatten(-1, (-1, 32)).amax(-1).double()
    assert (err <= 1.26).all() and (err.pow(2).mean() < 0.1)
    assert ((d.double().abs() / (most / 8) - 1).abs() <= 2.0 ** -5).all()
