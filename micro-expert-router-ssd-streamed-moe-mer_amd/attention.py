"""The attention side of a layer, between its projections and its router:
norms and rotation of queries and keys, the append to a paged key/value
cache and attention over it, over mer_hip_qk_norm_rope / mer_hip_kv_append /
mer_hip_paged_attention.

They stand in for what the engine does on the host between a layer's dense
projections and its routed experts (transformer.rs, the paged KV of
block_pool.rs) so that the hidden state of moe_forward can stay on the device
from layer to layer.  Tensors are torch tensors on the current HIP device;
the work runs on the caller's current stream.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .errors import raise_for_status

# torch dtype -> mer_float_type
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 6}


def _enter(t: torch.Tensor) -> tuple[int, int]:
    """(device, current stream) for work on t, which must be on the current device."""
    dev = t.get_device()
    if dev < 0:
        raise ValueError("expected a device tensor")
    if dev != torch._C._cuda_getDevice():
        raise ValueError(f"tensors are on cuda:{dev}, the current device is cuda:{torch.cuda.current_device()}")
    _lib.ensure_init(dev)
    return dev, torch._C._cuda_getCurrentRawStream(dev)


def _flat(t: torch.Tensor | None, dtype: torch.dtype, n: int, dev: int, name: str) -> int:
    """Address of a contiguous tensor of n elements (None: 0)."""
    if t is None:
        return 0
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must have {n} elements side by side, got {tuple(t.shape)} strides {t.stride()}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
    return t.data_ptr()


def _rows(t: torch.Tensor, n: int, h: int, d: int, dtype: torch.dtype, dev: int, name: str) -> int:
    """Stride of the token axis of t, [n, h, d] with its heads side by side."""
    if t.shape != (n, h, d) or t.dtype != dtype:
        raise ValueError(f"{name} must be {(n, h, d)} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
    a, b, c = t.stride()
    if (d > 1 and c != 1) or (h > 1 and b != d):
        raise ValueError(f"the heads of {name} must lie side by side (strides {t.stride()})")
    return a if n > 1 else h * d


def _shape(t: torch.Tensor, name: str) -> torch.Size:
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return t.shape


def _new(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """An output like t (rows of heads side by side, which _rows has checked) without gaps."""
    return torch.empty_like(t, memory_format=torch.contiguous_format, dtype=dtype)


class PagedKvCache:
    """Keys and values of one layer in pages: k and v are
    [n_pages, n_kv_heads, page_size, head_dim] tensors, float16 or bfloat16.
    Slot s of the cache is place s % page_size of page s // page_size; which
    pages belong to which sequence is the caller's business (block tables).
    k and v are written in place; a cache over other tensors is another cache
    (wrap)."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device=None):
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        self._set(torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedKvCache":
        """A cache over the caller's own k and v tensors."""
        self = cls.__new__(cls)
        self._set(k, v)
        return self

    def _set(self, k: torch.Tensor, v: torch.Tensor) -> None:
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be alike: [n_pages, n_kv_heads, page_size, head_dim]")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("k and v must be contiguous")
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"a cache is float16 or bfloat16, got {k.dtype}")
        self._k, self._v = k, v
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self._desc = _lib.MerKvCache(k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], self.page_size, self.n_kv_heads,
                                     self.head_dim, self.n_pages)
        self._ref = ctypes.byref(self._desc)
        self.device = k.get_device()

    # The calls go by the addresses taken above, so these cannot be replaced.
    k = property(lambda self: self._k, doc="the keys")
    v = property(lambda self: self._v, doc="the values")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None,
                 inv_freq: torch.Tensor | None, *, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                 out_dtype: torch.dtype | None = None, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None):
    """Norm of each query and key head, x / sqrt(mean(x^2) + eps) * norm, and
    the position rotation, in one pass; returns (q_out, k_out).

    q, k       [tokens, heads, head_dim] float32 / float16 / bfloat16, rows any
               16-byte stride apart (slices of a packed projection); k may be None
    positions  int32 [tokens]; inv_freq float32 [rot_dim / 2], None = no rotation
    q_norm, k_norm  float32 [head_dim], None = no norm
    interleaved     pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)
    q_out, k_out    may be q and k themselves; else made, of out_dtype (default: q's)
    """
    dev, stream = _enter(q)
    n, h, d = _shape(q, "q")
    src = q.dtype
    dt = out_dtype if out_dtype is not None else src if q_out is None else q_out.dtype
    if dt not in _TYPES:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, got {dt}")
    q_stride = _rows(q, n, h, d, src, dev, "q")
    if q_out is None:
        q_out, qo_stride = _new(q, dt), h * d
    else:
        qo_stride = _rows(q_out, n, h, d, dt, dev, "q_out")
    kh = k_ptr = k_stride = ko_ptr = ko_stride = 0
    if k is not None:
        kh = _shape(k, "k")[1]
        k_ptr, k_stride = k.data_ptr(), _rows(k, n, kh, d, src, dev, "k")
        if k_out is None:
            k_out, ko_stride = _new(k, dt), kh * d
        else:
            ko_stride = _rows(k_out, n, kh, d, dt, dev, "k_out")
        ko_ptr = k_out.data_ptr()
    elif k_out is not None or k_norm is not None:
        raise ValueError("k_out and k_norm need k")
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    rc = _lib.lib().mer_hip_qk_norm_rope(
        _TYPES[src], _TYPES[dt], n, h, kh, d, q.data_ptr(), q_stride, k_ptr, k_stride,
        _flat(positions, torch.int32, n, dev, "positions"), _flat(inv_freq, torch.float32, rot // 2, dev, "inv_freq"),
        rot, interleaved, _flat(q_norm, torch.float32, d, dev, "q_norm"),
        _flat(k_norm, torch.float32, d, dev, "k_norm"), eps, q_out.data_ptr(), qo_stride, ko_ptr, ko_stride, stream)
    if rc:
        raise_for_status(rc)
    return q_out, k_out


def kv_append(cache: PagedKvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
              positions: torch.Tensor | None = None, inv_freq: torch.Tensor | None = None,
              k_norm: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False) -> None:
    """Rows of k and v to their slots of the cache, the keys normed and
    rotated on the way (each optional, as in qk_norm_rope).

    k, v    [tokens, n_kv_heads, head_dim] float32 / float16 / bfloat16
    slots   int64 [tokens], distinct; negative = padding, the row is skipped; a
            slot past the cache is skipped and recorded (take_device_status)
    """
    dev, stream = _enter(k)
    n, src = _shape(k, "k")[0], k.dtype
    kh, d = cache.n_kv_heads, cache.head_dim
    ks, vs = _rows(k, n, kh, d, src, dev, "k"), _rows(v, n, kh, d, src, dev, "v")
    if cache.device != dev:
        raise ValueError(f"the cache is on cuda:{cache.device}, expected cuda:{dev}")
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    rc = _lib.lib().mer_hip_kv_append(
        cache._ref, _TYPES[src], n, k.data_ptr(), ks, v.data_ptr(), vs, _flat(slots, torch.int64, n, dev, "slots"),
        _flat(positions, torch.int32, n, dev, "positions"), _flat(inv_freq, torch.float32, rot // 2, dev, "inv_freq"),
        rot, interleaved, _flat(k_norm, torch.float32, d, dev, "k_norm"), eps, stream)
    if rc:
        raise_for_status(rc)


def paged_attention(cache: PagedKvCache, q: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor,
                    kv_len: torch.Tensor, *, max_q_len: int = 0, max_kv_len: int = 0, scale: float | None = None,
                    window: int = 0, sinks: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's new tokens over its pages; decode steps,
    prompt chunks and mixes of both in one call.

    q            [tokens, n_heads, head_dim] of the cache's type
    block_table  int32 [n_seqs, pages]: page ids of each sequence, in order
    q_start      int32 [n_seqs + 1]: sequence s has rows q_start[s] .. q_start[s + 1]
    kv_len       int32 [n_seqs]: its keys in the cache, the new tokens' own among
                 them; the rows are the last positions
    max_q_len, max_kv_len  what to lay the call out for (0 = unknown); results
                 do not depend on them
    scale        of q . k, default 1 / sqrt(head_dim)
    window       keys a row sees, itself included; 0 = all
    sinks        float32 [n_heads]: a logit per head that adds no value
    out          like q, or q itself; made with zeros in rows of no sequence when None
    """
    dev, stream = _enter(q)
    n, h, d = _shape(q, "q")
    if d != cache.head_dim or q.dtype != cache.k.dtype or cache.device != dev:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} on cuda:{dev} does not go with a cache of head_dim "
                         f"{cache.head_dim}, {cache.k.dtype} on cuda:{cache.device}")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [n_seqs, pages]")
    seqs, width = block_table.shape
    if out is None:
        out, out_stride = torch.zeros((n, h, d), dtype=q.dtype, device=q.device), h * d
    else:
        out_stride = _rows(out, n, h, d, q.dtype, dev, "out")
    if window < 0 or max_q_len < 0 or max_kv_len < 0:
        raise ValueError("window, max_q_len and max_kv_len must not be negative")
    if scale is not None and ctypes.c_float(scale).value == 0:  # which the entry point takes for the default
        raise ValueError(f"the scale {scale} is zero in float32")
    rc = _lib.lib().mer_hip_paged_attention(
        cache._ref, seqs, n, h, q.data_ptr(), _rows(q, n, h, d, q.dtype, dev, "q"),
        _flat(block_table, torch.int32, seqs * width, dev, "block_table"), width,
        _flat(q_start, torch.int32, seqs + 1, dev, "q_start"), _flat(kv_len, torch.int32, seqs, dev, "kv_len"),
        max_q_len, max_kv_len, 0.0 if scale is None else scale, min(window, 0xffffffff),
        _flat(sinks, torch.float32, h, dev, "sinks"), out.data_ptr(), out_stride, stream)
    if rc:
        raise_for_status(rc)
    return out
