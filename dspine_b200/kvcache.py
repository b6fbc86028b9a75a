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
_INDEX = {torch.int32: 0, torch.int64: 1}
_ROWS = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


def _check(cond, msg):
    if not cond:
        raise ValueError(msg)


# the cheap forms of torch.cuda.current_device() and current_stream(index).cuda_stream
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


def launch(fn, dev, *args):
    """Call the C entry `fn` with the current stream of `dev` as its last argument, `dev` made current for
    the launch where it is not."""
    index = dev.index
    now = _current_device()
    if now == index:
        _lib.call(fn, *args, _raw_stream(index))
        return
    torch.cuda.set_device(index)
    try:
        _lib.call(fn, *args, _raw_stream(index))
    finally:
        torch.cuda.set_device(now)


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
    shape, s = k_cache.shape, k_cache.stride()
    dtype = _CACHE.get(k_cache.dtype)
    dev = k_cache.device
    if dtype is None or len(shape) != 3 or v_cache.shape != shape or v_cache.dtype != k_cache.dtype or v_cache.stride() != s or v_cache.device != dev:
        _check(k_cache.dim() == 3 and v_cache.shape == shape, "k_cache and v_cache must be [slots, heads, dim]")
        _check(dtype is not None and v_cache.dtype == k_cache.dtype,
               f"a KV cache holds bf16, fp16 or e4m3 rows, got {k_cache.dtype}, {v_cache.dtype}")
        _check(v_cache.device == dev, "the cache must be on one device")
        _check(False, "k_cache and v_cache must have the same strides and contiguous rows")
    slots, heads, dim = shape
    slot_stride, head_stride, one = s
    step = 16 if dtype == 3 else 8
    if dim % 16 or not dim or one != 1 or slots < 1 or heads < 1:
        _check(dim % 16 == 0 and dim >= 16, "dim must be a multiple of 16")
        _check(one == 1, "k_cache and v_cache must have the same strides and contiguous rows")
        _check(False, "the cache has no slots")
    # a dimension of one element may carry any stride: it is never stepped over
    if heads == 1:
        head_stride = dim
    if slots == 1:
        slot_stride = heads * head_stride
    if slot_stride < dim or slot_stride % step or head_stride < dim or head_stride % step:
        _check(False, "the cache's rows must be 16-byte aligned and not overlap")
    if dtype != 3:
        _check(k_scale is None and v_scale is None, "only an e4m3 cache has scales")
        return _lib.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), None, None, slots, slot_stride, head_stride, heads, heads, dim,
                            dtype)
    _check(k_scale is not None and v_scale is not None, "an e4m3 cache needs k_scale and v_scale")
    for x in (k_scale, v_scale):
        if x.shape != (slots, heads) or x.dtype != torch.float32 or x.device != dev:
            _check(False, "k_scale and v_scale must be fp32 [slots, heads]")
    ss = k_scale.stride()
    if ss != v_scale.stride() or (heads > 1 and ss[1] != 1):
        _check(heads == 1 or (ss[1] == 1 and v_scale.stride(1) == 1), "a slot's scales must be adjacent")
        _check(slots == 1, "k_scale and v_scale must have the same strides")
    scale_stride = ss[0] if slots > 1 else heads
    _check(scale_stride >= heads, "the scales of two slots overlap")
    return _lib.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), slots, slot_stride, head_stride,
                        scale_stride, heads, dim, dtype)


def _slots(slots, dev):
    if slots.dim() != 1 or slots.dtype not in _INDEX or slots.device != dev or not slots.is_contiguous():
        _check(slots.dim() == 1, "slots must be [tokens]")
        _check(slots.dtype in _INDEX and slots.device == dev, "slots must be int32 or int64 on the cache's device")
        _check(False, "slots must be contiguous")
    return _INDEX[slots.dtype]


def check_err(err, dev):
    _check(err is None or (err.dtype == torch.int32 and err.numel() == 1 and err.device == dev), "err must be one int32 on the cache's device")


def write_kv(k, v, k_cache, v_cache, slots, *, k_scale=None, v_scale=None, err=None):
    """Store token n's rows k[n], v[n] ([tokens, heads, dim]) at slot slots[n] of the cache.

    bf16 and fp16 rows go into a cache of their own type as they are; rows of bf16, fp16 or fp32
    go into an e4m3 cache as codes, with their scale amax / 448 in k_scale and v_scale.  Rows may
    be views of a wider projection (any token and head strides of 16-byte steps).  A negative slot
    is skipped; one past the cache is skipped and sets bit 0 of `err` (int32 [1], optional).  The
    slots of one call should differ: of tokens that share one, any may be kept, or a mixture.  k and v
    must not be views of the cache itself."""
    c = describe(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    shape = k.shape
    _check(len(shape) == 3 and v.shape == shape and shape[1] == c.heads and shape[2] == c.dim, "k and v must be [tokens, heads, dim] as the cache")
    dtype = _ROWS.get(k.dtype)
    if dtype is None or v.dtype != k.dtype:
        _check(False, f"rows must be bf16, fp16 or fp32, got {k.dtype}, {v.dtype}")
    _check(c.dtype == 3 or c.dtype == dtype, "a cache that is not e4m3 takes rows of its own type")
    _check(k.device == dev and v.device == dev, "tensors must be on one CUDA device")
    (kt, kh, k1), (vt, vh, v1) = k.stride(), v.stride()
    _check(k1 == 1 and v1 == 1, "rows must be contiguous")
    _check(c.dim <= 256, "dim must be at most 256")
    is64 = _slots(slots, dev)
    n = shape[0]
    _check(slots.shape[0] == n, "slots must be [tokens]")
    if err is not None:
        check_err(err, dev)
    _check(dev.type == "cuda", "the cache must be on a CUDA device")
    if n == 0:
        return
    if n == 1:
        kt = vt = 0
    if c.heads == 1:
        kh = vh = 0
    launch("dsv_kv_write", dev, n, dtype, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, slots.data_ptr(), is64, c,
           None if err is None else err.data_ptr())


def read_kv(k_cache, v_cache, slots, *, k_scale=None, v_scale=None, dtype=torch.bfloat16, out=None, err=None):
    """(k, v) [tokens, heads, dim] of `dtype` (bf16, fp16 or fp32): the rows of slots[n], code *
    scale in fp32 rounded once.  A negative slot gives zeros; one past the cache too, and sets
    bit 0 of `err`.  `out` gives the two tensors to fill."""
    c = describe(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _check(c.dim <= 256, "dim must be at most 256")
    is64 = _slots(slots, dev)
    if err is not None:
        check_err(err, dev)
    n = slots.shape[0]
    shape = (n, c.heads, c.dim)
    if out is None:
        code = _ROWS.get(dtype)
        if code is None:
            _check(False, f"rows are read as bf16, fp16 or fp32, got {dtype}")
        k = torch.empty(shape, dtype=dtype, device=dev)
        v = torch.empty_like(k)
    else:
        k, v = out
        code = _ROWS.get(k.dtype)
        for x in out:
            _check(code is not None and x.shape == shape and x.dtype == k.dtype and x.is_contiguous() and x.device == dev,
                   "out must be two contiguous [tokens, heads, dim] tensors of bf16, fp16 or fp32")
    _check(dev.type == "cuda", "the cache must be on a CUDA device")
    if n:
        launch("dsv_kv_read", dev, n, slots.data_ptr(), is64, c, code, k.data_ptr(), v.data_ptr(), None if err is None else err.data_ptr())
    return k, v
