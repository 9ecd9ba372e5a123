"""Refusals of the attention-side entry points: arguments are checked before
any device work, so they are tested without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 255) & ~255  # an aligned address that nothing reads


@pytest.fixture
def abi(mer):
    return mer._lib


def cache(abi, **kw):
    f = dict(k=P, v=P, type=1, page_size=16, n_kv_heads=2, head_dim=64, n_pages=4)
    f.update(kw)
    return ctypes.byref(abi.MerKvCache(*f.values()))


def norm_rope(abi, **kw):
    f = dict(in_type=1, out_type=1, n=4, h=4, kv=2, d=64, q=P, qs=256, k=P, ks=128, pos=P,
             freq=P, rot=64, interleaved=0, qn=P, kn=P, eps=1e-6, qo=P, qos=256, ko=P, kos=128,
             stream=None)
    f.update(kw)
    return abi.lib().mer_hip_qk_norm_rope(*f.values())


def append(abi, c=None, **kw):
    f = dict(cache=c if c is not None else cache(abi), in_type=1, n=4, k=P, ks=128, v=P, vs=128, slots=P, pos=P,
             freq=P, rot=64, interleaved=0, kn=P, eps=1e-6, stream=None)
    f.update(kw)
    return abi.lib().mer_hip_kv_append(*f.values())


def attention(abi, c=None, **kw):
    f = dict(cache=c if c is not None else cache(abi), seqs=2, n=4, h=4, q=P, qs=256, table=P, width=4, start=P,
             lens=P, mq=0, mk=0, scale=0.0, window=0, sinks=None, out=P, os=256, stream=None)
    f.update(kw)
    return abi.lib().mer_hip_paged_attention(*f.values())


def test_good_arguments_get_as_far_as_the_device(abi):
    expected = (abi.Status.NOT_INITIALIZED,)
    if torch.cuda.is_available():
        pytest.skip("would run on the GPU")
    for call in (norm_rope, append, attention):
        assert call(abi) in expected
        assert call(abi, n=0) == 0  # nothing to do
    assert attention(abi, seqs=0) == 0


@pytest.mark.parametrize("change,status", [
    (dict(in_type=4), "UNSUPPORTED_DTYPE"), (dict(out_type=5), "UNSUPPORTED_DTYPE"),
    (dict(d=0), "INVALID_LAYOUT"), (dict(d=60), "INVALID_LAYOUT"), (dict(d=264), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(h=0, kv=0), "INVALID_LAYOUT"), (dict(h=4096), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(n=(1 << 24) + 1), "SHAPE_EXCEEDS_WORKSPACE"), (dict(n=1 << 24), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(q=None), "INVALID_LAYOUT"), (dict(ko=None), "INVALID_LAYOUT"), (dict(pos=None), "INVALID_LAYOUT"),
    (dict(q=P + 2), "MISALIGNED"), (dict(qs=260), "MISALIGNED"), (dict(qs=248), "INVALID_LAYOUT"),
    (dict(kos=0), "INVALID_LAYOUT"), (dict(qn=P + 4), "MISALIGNED"), (dict(ks=1 << 41), "INVALID_LAYOUT"),
    (dict(pos=P + 2), "MISALIGNED"), (dict(eps=-1e-6), "INVALID_LAYOUT"), (dict(eps=float("nan")), "INVALID_LAYOUT"),
    (dict(eps=float("inf"), qn=0), "INVALID_LAYOUT"),
])
def test_norm_rope_refuses(abi, change, status):
    assert norm_rope(abi, **change) == abi.Status[status]
    assert abi.last_error()[0] == abi.Status[status] and abi.last_error()[1]


@pytest.mark.parametrize("rot,freq,status", [(4, P, "INVALID_LAYOUT"), (12, P, "INVALID_LAYOUT"),
                                             (72, P, "INVALID_LAYOUT"), (64, 0, "INVALID_LAYOUT"),
                                             (64, P + 8, "MISALIGNED")])
def test_rotation_refused(abi, rot, freq, status):
    assert norm_rope(abi, freq=freq, rot=rot) == abi.Status[status]
    assert append(abi, freq=freq, rot=rot) == abi.Status[status]


@pytest.mark.parametrize("change,status", [
    (dict(k=0), "INVALID_LAYOUT"), (dict(v=P + 8), "MISALIGNED"), (dict(type=0), "UNSUPPORTED_DTYPE"),
    (dict(type=5), "UNSUPPORTED_DTYPE"), (dict(page_size=4), "INVALID_LAYOUT"), (dict(page_size=24), "INVALID_LAYOUT"),
    (dict(page_size=8192), "INVALID_LAYOUT"), (dict(n_kv_heads=0), "INVALID_LAYOUT"),
    (dict(head_dim=68), "INVALID_LAYOUT"), (dict(head_dim=512), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(n_pages=0), "INVALID_LAYOUT"), (dict(n_pages=1 << 31), "INVALID_LAYOUT"),
])
def test_cache_refused(abi, change, status):
    assert append(abi, cache(abi, **change)) == abi.Status[status]
    assert attention(abi, cache(abi, **change)) == abi.Status[status]


def test_null_cache_refused(abi):
    assert append(abi, cache=None) == abi.Status.INVALID_LAYOUT
    assert attention(abi, cache=None) == abi.Status.INVALID_LAYOUT


@pytest.mark.parametrize("change,status", [
    (dict(in_type=3), "UNSUPPORTED_DTYPE"), (dict(k=None), "INVALID_LAYOUT"), (dict(v=P + 4), "MISALIGNED"),
    (dict(ks=132), "MISALIGNED"), (dict(vs=120), "INVALID_LAYOUT"), (dict(slots=None), "INVALID_LAYOUT"),
    (dict(pos=None), "INVALID_LAYOUT"), (dict(n=1 << 25), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(slots=P + 4), "MISALIGNED"), (dict(pos=P + 1), "MISALIGNED"), (dict(eps=-1.0), "INVALID_LAYOUT"),
])
def test_append_refuses(abi, change, status):
    assert append(abi, **change) == abi.Status[status]


@pytest.mark.parametrize("change,status", [
    (dict(h=3), "INVALID_LAYOUT"), (dict(h=0), "INVALID_LAYOUT"), (dict(seqs=(1 << 20) + 1), "SHAPE_EXCEEDS_WORKSPACE"),
    (dict(width=(1 << 26) + 1), "SHAPE_EXCEEDS_WORKSPACE"), (dict(q=None), "INVALID_LAYOUT"),
    (dict(qs=250), "MISALIGNED"), (dict(out=P + 6), "MISALIGNED"), (dict(table=None), "INVALID_LAYOUT"),
    (dict(start=P + 2), "MISALIGNED"), (dict(lens=P + 1), "MISALIGNED"), (dict(table=P + 2), "MISALIGNED"),
    (dict(start=None), "INVALID_LAYOUT"), (dict(lens=None), "INVALID_LAYOUT"), (dict(n=1 << 25), "SHAPE_EXCEEDS_WORKSPACE"),
])
def test_attention_refuses(abi, change, status):
    assert attention(abi, **change) == abi.Status[status]


@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_attention_refuses_a_scale(abi, scale):
    assert attention(abi, scale=scale) == abi.Status.INVALID_LAYOUT


def test_python_refusals(mer):
    with pytest.raises(ValueError):
        mer.qk_norm_rope(torch.zeros(1, 1, 64), None, None, None)  # not on a device
    with pytest.raises(TypeError):
        mer.PagedKvCache.wrap(torch.zeros(1, 1, 8, 64), torch.zeros(1, 1, 8, 64))
    with pytest.raises(ValueError):
        mer.PagedKvCache.wrap(torch.zeros(1, 1, 8, 64).half(), torch.zeros(2, 1, 8, 64).half())
    with pytest.raises(ValueError):
        mer.PagedKvCache.wrap(torch.zeros(1, 1, 8, 128).half()[..., ::2], torch.zeros(1, 1, 8, 64).half())


def test_the_tensors_of_a_cache_cannot_be_replaced(mer):
    """A call goes by the addresses of the cache's own tensors; one over other
    tensors is another cache."""
    k, v = torch.zeros(2, 1, 8, 64).half(), torch.ones(2, 1, 8, 64).half()
    cache = mer.PagedKvCache.wrap(k, v)
    for name in ("k", "v"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros(2, 1, 8, 64).half())
    assert cache.k is k and cache.v is v and (cache._desc.k, cache._desc.v) == (k.data_ptr(), v.data_ptr())


def test_attention_refuses_a_scale_that_overflows_in_base_2(abi):
    """scale * log2(e), which the kernels multiply with, has to be finite too."""
    good, bad = 2.35e38, 2.36e38  # 3.4028e38 / log2(e) = 2.3587e38
    expected = abi.Status.NOT_INITIALIZED
    for sign in (1, -1):
        assert attention(abi, scale=sign * bad) == abi.Status.INVALID_LAYOUT
        if not torch.cuda.is_available():
            assert attention(abi, scale=sign * good) == expected


@pytest.mark.parametrize("h,kv", [((1 << 64) - 1, 2), (3, (1 << 64) - 1), (1 << 63, 1 << 63)])
def test_norm_rope_refuses_heads_whose_sum_wraps(abi, h, kv):
    assert norm_rope(abi, n=1, h=h, kv=kv) == abi.Status.SHAPE_EXCEEDS_WORKSPACE
