"""Host API of the slot-addressed KV cache (C ABI: dsv_kv_write, dsv_kv_read).

The cache is what the KV slots of the accept step point into (`out_cache_loc`, page size 1 or
more): K and V tensors [slots, heads, dim] that hold the rows as they are (bf16 or fp16), or e4m3
codes with one fp32 scale per (slot, head), quantised by the rule of the FP8 retrieval head
(`layers.fp8.coarse.quantize_rows`) applied to each head's row.  `write_kv` stores the rows of
new tokens, `read_kv` gathers rows back, `attention.tree_attention` reads the cache in place.
Argument errors raise ValueError before anything is launched.
"""

from __future__ import annotations

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
_CACHE = {torch.bfloat16: 0, torch.float16: 2, E4M3: 3}
_ROWS = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


def _check(cond, msg):
    if not cond:
        raise ValueError(msg)


class on_device:
    """The tensors' device made current for a launch (nothing to do where it is already)."""

    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index
        self.before = None

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self.index:
            self.before = now
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.before is not None:
            torch.cuda.set_device(self.before)


def allocate_kv(slots, heads, dim, *, dtype=torch.bfloat16, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of `slots` slots, zeroed; the scales (ones) are None
    unless dtype is float8_e4m3fn."""
    _check(dtype in _CACHE, f"a KV cache holds bf16, fp16 or e4m3 rows, got {dtype}")
    _check(dim % 16 == 0 and 16 <= dim <= 256, "dim must be a multiple of 16 in [16, 256]")
    shape = (int(slots), int(heads), int(dim))
    if dtype is not E4M3:
        return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), None, None
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(E4M3) for _ in range(2))
    ks, vs = (torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
    return k, v, ks, vs


def describe(k_cache, v_cache, k_scale, v_scale):
    """The C view of a cache (_lib.KvCache), its tensors checked."""
    _check(k_cache.dim() == 3 and k_cache.shape == v_cache.shape, "k_cache and v_cache must be [slots, heads, dim]")
    dtype = _CACHE.get(k_cache.dtype)
    _check(dtype is not None and v_cache.dtype == k_cache.dtype, f"a KV cache holds bf16, fp16 or e4m3 rows, got {k_cache.dtype}, {v_cache.dtype}")
    slots, heads, dim = k_cache.shape
    s = k_cache.stride()
    _check(s == v_cache.stride() and (s[2] == 1 or dim == 1), "k_cache and v_cache must have the same strides and contiguous rows")
    dev = k_cache.device
    _check(v_cache.device == dev, "the cache must be on one device")
    _check(dim % 16 == 0 and dim >= 16, "dim must be a multiple of 16")
    _check(slots >= 1 and heads >= 1, "the cache has no slots")
    step = 16 if dtype == 3 else 8
    _check((slots == 1 or (s[0] >= dim and s[0] % step == 0)) and (heads == 1 or (s[1] >= dim and s[1] % step == 0)),
           "the cache's rows must be 16-byte aligned and not overlap")
    # a dimension of one element may carry any stride: it is never stepped over
    slot_stride = s[0] if slots > 1 else max(heads * dim, dim)
    head_stride = s[1] if heads > 1 else dim
    if dtype == 3:
        _check(k_scale is not None and v_scale is not None, "an e4m3 cache needs k_scale and v_scale")
        for x in (k_scale, v_scale):
            _check(x.shape == (slots, heads) and x.dtype == torch.float32 and x.device == dev, "k_scale and v_scale must be fp32 [slots, heads]")
            _check(heads == 1 or x.stride(1) == 1, "a slot's scales must be adjacent")
        _check(k_scale.stride(0) == v_scale.stride(0) or slots == 1, "k_scale and v_scale must have the same strides")
        scale_stride = k_scale.stride(0) if slots > 1 else heads
        _check(scale_stride >= heads, "the scales of two slots overlap")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        _check(k_scale is None and v_scale is None, "only an e4m3 cache has scales")
        ks = vs = None
        scale_stride = heads
    return _lib.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), ks, vs, slots, slot_stride, head_stride, scale_stride,
                        heads, dim, dtype)


def _slots(slots, n, dev):
    _check(slots.dim() == 1 and (n is None or slots.shape[0] == n), "slots must be [tokens]")
    _check(slots.dtype in (torch.int32, torch.int64) and slots.device == dev, "slots must be int32 or int64 on the cache's device")
    _check(slots.shape[0] <= 1 or slots.stride(0) == 1, "slots must be contiguous")
    return int(slots.dtype == torch.int64)


def check_err(err, dev):
    _check(err is None or (err.dtype == torch.int32 and err.numel() == 1 and err.device == dev), "err must be one int32 on the cache's device")


def write_kv(k, v, k_cache, v_cache, slots, *, k_scale=None, v_scale=None, err=None):
    """Store token n's rows k[n], v[n] ([tokens, heads, dim]) at slot slots[n] of the cache.

    bf16 and fp16 rows go into a cache of their own type as they are; rows of bf16, fp16 or fp32
    go into an e4m3 cache as codes, with their scale amax / 448 in k_scale and v_scale.  Rows may
    be views of a wider projection (any token and head strides of 16-byte steps).  A negative slot
    is skipped; one past the cache is skipped and sets bit 0 of `err` (int32 [1], optional).  The
    slots of one call should differ: of tokens that share one, any may be kept, or a mixture."""
    c = describe(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _check(k.dim() == 3 and v.dim() == 3 and k.shape == v.shape and k.shape[1:] == k_cache.shape[1:],
           "k and v must be [tokens, heads, dim] as the cache")
    dtype = _ROWS.get(k.dtype)
    _check(dtype is not None and v.dtype == k.dtype, f"rows must be bf16, fp16 or fp32, got {k.dtype}, {v.dtype}")
    _check(c.dtype == 3 or c.dtype == dtype, "a cache that is not e4m3 takes rows of its own type")
    _check(k.device == dev and v.device == dev, "tensors must be on one CUDA device")
    _check(k.stride(2) == 1 and v.stride(2) == 1, "rows must be contiguous")
    _check(c.dim <= 256, "dim must be at most 256")
    is64 = _slots(slots, k.shape[0], dev)
    check_err(err, dev)
    _check(dev.type == "cuda", "the cache must be on a CUDA device")
    n = k.shape[0]
    if n == 0:
        return
    with on_device(dev) as stream:
        _lib.call("dsv_kv_write", n, dtype, k.data_ptr(), k.stride(0) if n > 1 else 0, k.stride(1) if c.heads > 1 else 0,
                  v.data_ptr(), v.stride(0) if n > 1 else 0, v.stride(1) if c.heads > 1 else 0, slots.data_ptr(), is64,
                  c, _lib.ptr(err), stream)


def read_kv(k_cache, v_cache, slots, *, k_scale=None, v_scale=None, dtype=torch.bfloat16, out=None, err=None):
    """(k, v) [tokens, heads, dim] of `dtype` (bf16, fp16 or fp32): the rows of slots[n], code *
    scale in fp32 rounded once.  A negative slot gives zeros; one past the cache too, and sets
    bit 0 of `err`.  `out` gives the two tensors to fill."""
    c = describe(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _check(c.dim <= 256, "dim must be at most 256")
    is64 = _slots(slots, None, dev)
    check_err(err, dev)
    n = slots.shape[0]
    shape = (n, c.heads, c.dim)
    if out is None:
        _check(dtype in _ROWS, f"rows are read as bf16, fp16 or fp32, got {dtype}")
        out = (torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev))
    k, v = out
    for x in out:
        _check(x.shape == shape and x.dtype in _ROWS and x.dtype == k.dtype and x.is_contiguous() and x.device == dev,
               "out must be two contiguous [tokens, heads, dim] tensors of bf16, fp16 or fp32")
    _check(dev.type == "cuda", "the cache must be on a CUDA device")
    if n:
        with on_device(dev) as stream:
            _lib.call("dsv_kv_read", n, slots.data_ptr(), is64, c, _ROWS[k.dtype], k.data_ptr(), v.data_ptr(),
                      _lib.ptr(err), stream)
    return k, v
