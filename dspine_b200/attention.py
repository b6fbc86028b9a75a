"""Host API of the drafted tokens' attention over the KV cache (C ABI: dsv_tree_attention).

`tree_attention` is the attention of a verification step: every request's drafted tokens, a chain
or a tree, attend over its cached context and over their own ancestors, in place over a paged,
slot-addressed cache (`kvcache`).  One drafted token per request is ordinary decoding.
`tree_mask` turns parents into the ancestor bits that it and `accept.accept_tree` take.
Argument errors raise ValueError before anything is launched.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .kvcache import _check, check_err, describe, on_device

MAX_DIM = 128
MAX_NODES = 64
_DTYPES = {torch.bfloat16: 0, torch.float16: 2}


def tree_mask(parents):
    """int64 ancestor bits from parents [..., nodes] (nodes <= 64; -1 for a root, which comes
    first; parents before children): bit j of node i is set where j is i or an ancestor of i."""
    _check(parents.dim() >= 1 and parents.shape[-1] <= MAX_NODES, f"a draft tree has at most {MAX_NODES} nodes")
    _check(not parents.is_floating_point(), "parents must be integers")
    n = parents.shape[-1]
    up = parents.long()
    mask = torch.ones_like(up) << torch.arange(n, device=up.device)
    for _ in range(max(1, n - 1).bit_length()):  # pointer doubling: 2^k ancestors after k steps
        at = up.clamp(min=0)
        mask = torch.where(up >= 0, mask | mask.gather(-1, at), mask)
        up = torch.where(up >= 0, up.gather(-1, at), up)
    return mask


_sizes: dict = {}


def workspace_bytes(q_heads, kv_heads, dim, width) -> int:
    """Device scratch of one call (partial results of split contexts)."""
    key = (q_heads, kv_heads, dim, width)
    n = _sizes.get(key)
    if n is None:
        size = ctypes.c_size_t()
        _lib.call("dsv_tree_attention_workspace_size", q_heads, kv_heads, dim, width, ctypes.byref(size))
        n = _sizes[key] = int(size.value)
    return n


def tree_attention(q, k_cache, v_cache, page_table, kv_lens, *, page_size=1, q_indptr=None, max_width=None,
                   tree_mask=None, scale=None, k_scale=None, v_scale=None, out=None, lse=None,
                   return_lse=False, workspace=None, err=None):
    """Attention of drafted tokens over a paged KV cache.

    q [rows, q_heads, dim] bf16 or fp16; k_cache, v_cache [slots, kv_heads, dim] of q's type, or
    e4m3 with k_scale, v_scale [slots, kv_heads]; dim a multiple of 16 up to 128, q_heads a
    multiple of kv_heads.  Request b owns rows [q_indptr[b], q_indptr[b+1]) (int32 [B+1]; None:
    rows / B each) and kv_lens[b] (int32) cached positions, its drafted tokens the last of them:
    their K and V are written before the call.  Position p is slot page_table[b, p // page_size]
    * page_size + p % page_size (page_table int32 [B, pages]).

    Row i of a request sees every position before its drafted tokens, and drafted token j where
    bit j of tree_mask[row] (int64 [rows]) is set, or without a tree_mask where j <= i.  The result is
    softmax(scale q.k) v (scale 1/sqrt(dim) unless given), zeros for a row that sees nothing;
    `return_lse` adds the fp32 [rows, q_heads] logsumexp.  Rows of no request are left as they were.

    max_width: a bound on the rows of a request, by which the work is laid out (results do not
    depend on it); default 64 with a tree_mask, else all rows.  A tree has at most 64 nodes.
    workspace: uint8 scratch of `workspace_bytes` (allocated for the call unless given); calls that may
    overlap need one each.  err (int32 [1], optional) collects bit 1: a page outside the cache or
    a length past the page table (those positions are unseen), bit 2: a wait that timed out.  A
    masked position's K may hold anything; V of positions that some row of the request sees
    reaches the rows that see it alone, infinities and NaN included."""
    c = describe(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    _check(q.dim() == 3 and q.dtype in _DTYPES, "q must be bf16 or fp16 [rows, q_heads, dim]")
    rows, q_heads, dim = q.shape
    dtype = _DTYPES[q.dtype]
    _check(dim == c.dim and dim <= MAX_DIM, f"q and the cache must have one dim, at most {MAX_DIM}")
    _check(q_heads >= 1 and q_heads % c.heads == 0 and q_heads <= 4096 * c.heads,
           "q_heads must be a multiple of the cache's heads, at most 4096 of them each")
    _check(c.dtype == 3 or c.dtype == dtype, "the cache must have q's type or be e4m3")
    _check(page_table.dim() == 2 and page_table.dtype == torch.int32, "page_table must be int32 [requests, pages]")
    batch, pages = page_table.shape
    _check(pages <= 1 or page_table.stride(1) == 1, "page_table's rows must be contiguous")
    _check(batch <= 1 or page_table.stride(0) >= pages, "page_table's rows overlap")
    _check(kv_lens.shape == (batch,) and kv_lens.dtype == torch.int32 and (batch <= 1 or kv_lens.stride(0) == 1),
           "kv_lens must be contiguous int32 [requests]")
    page_size = int(page_size)
    _check(page_size >= 1 and c.slots % page_size == 0, "the cache must hold whole pages of page_size slots")
    if q_indptr is None:
        _check(batch > 0 and rows % batch == 0 or rows == 0, "without q_indptr every request has the same number of rows")
        width = max(1, rows // max(batch, 1))
        _check(tree_mask is None or width <= MAX_NODES, f"a draft tree has at most {MAX_NODES} nodes")
    else:
        _check(q_indptr.shape == (batch + 1,) and q_indptr.dtype == torch.int32 and (batch < 1 or q_indptr.stride(0) == 1),
               "q_indptr must be contiguous int32 [requests + 1]")
        width = (max(rows, 1) if tree_mask is None else MAX_NODES) if max_width is None else int(max_width)
        _check(width >= 1, "max_width must be at least 1")
        _check(q_indptr.device == dev, "tensors must be on one CUDA device")
    if tree_mask is not None:
        _check(tree_mask.shape == (rows,) and tree_mask.dtype == torch.int64 and (rows <= 1 or tree_mask.stride(0) == 1),
               "tree_mask must be contiguous int64 [rows]")
        _check(tree_mask.device == dev, "tensors must be on one CUDA device")
    _check(q.device == dev and page_table.device == dev and kv_lens.device == dev, "tensors must be on one CUDA device")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    _check(0.0 < scale < 3.4e38, "scale must be positive and finite")
    if out is None:
        out = torch.empty((rows, q_heads, dim), dtype=q.dtype, device=dev)
    _check(out.shape == q.shape and out.dtype == q.dtype and out.device == dev, "out must be like q")
    for x in (q, out):
        _check(rows == 0 or x.stride(2) == 1, "rows of q and out must be contiguous")
    _check((rows <= 1 or out.stride(0) >= dim) and (q_heads == 1 or out.stride(1) >= dim), "the rows of out overlap")
    if lse is None and return_lse:
        lse = torch.empty((rows, q_heads), dtype=torch.float32, device=dev)
    _check(lse is None or (lse.shape == (rows, q_heads) and lse.dtype == torch.float32 and lse.is_contiguous() and lse.device == dev),
           "lse must be contiguous fp32 [rows, q_heads]")
    check_err(err, dev)
    _check(dev.type == "cuda", "tensors must be on a CUDA device")
    if rows and batch:
        need = workspace_bytes(q_heads, c.heads, dim, width)
        with on_device(dev) as stream:
            if workspace is None:
                workspace = torch.empty(need, dtype=torch.uint8, device=dev)
            _check(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need and workspace.device == dev,
                   f"workspace must be {need} bytes (uint8) on the cache's device")
            _lib.call("dsv_tree_attention", batch, rows, q_heads, dtype, q.data_ptr(), q.stride(0) if rows > 1 else 0,
                      q.stride(1) if q_heads > 1 else 0, c, page_table.data_ptr() if pages else None,
                      page_table.stride(0) if batch > 1 else pages, pages, page_size, kv_lens.data_ptr(), _lib.ptr(q_indptr), width,
                      _lib.ptr(tree_mask), scale, out.data_ptr(), out.stride(0) if rows > 1 else 0,
                      out.stride(1) if q_heads > 1 else 0, _lib.ptr(lse), _lib.ptr(err), workspace.data_ptr() if need else None,
                      workspace.numel(), stream)
    return (out, lse) if return_lse else out
