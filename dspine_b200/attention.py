"""Host API of the drafted tokens' attention over the KV cache (C ABI: dsv_tree_attention).

`tree_attention` is the attention of a verification step: every request's drafted tokens, a chain
or a tree, attend over its cached context and over their own ancestors, in place over a paged,
slot-addressed cache (`kvcache`).  One drafted token per request is ordinary decoding.
`tree_mask` turns parents into the ancestor bits that it and `accept.accept_tree` take.
Argument errors raise ValueError before anything is launched.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from .kvcache import _check, check_err, describe, launch

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


@functools.lru_cache(maxsize=64)
def workspace_bytes(q_heads, kv_heads, dim, width) -> int:
    """Device scratch of one call (partial results of split contexts)."""
    size = ctypes.c_size_t()
    _lib.call("dsv_tree_attention_workspace_size", q_heads, kv_heads, dim, width, ctypes.byref(size))
    return int(size.value)


def tree_attention(q, k_cache, v_cache, page_table, kv_lens, *, page_size=1, q_indptr=None, max_width=None,
                   tree_mask=None, scale=None, k_scale=None, v_scale=None, out=None, lse=None,
                   return_lse=False, workspace=None, err=None):
    """Attention of drafted tokens over a paged KV cache.

    q [rows, q_heads, dim] bf16 or fp16; k_cache, v_cache [slots, kv_heads, dim] of q's type, or
    e4m3 with k_scale, v_scale [slots, kv_heads]; dim a multiple of 16 up to 128, q_heads a
    multiple of kv_heads.  Request b owns rows [q_indptr[b], q_indptr[b+1]) (int32 [B+1]; None:
    rows / B each) and kv_lens[b] (int32) cached positions, its drafted tokens the last of them:
    their K and V are written before the call.  Position p is slot page_table[b, p // page_size]
    * page_size + p % page_size (page_table int32 [B, pages], pages * page_size < 2^31 - 255).

    Row i of a request sees every position before its drafted tokens, and drafted token j where
    bit j of tree_mask[row] (int64 [rows]) is set, or without a tree_mask where j <= i.  The result is
    softmax(scale q.k) v (scale 1/sqrt(dim) unless given), zeros for a row that sees nothing (or scores
    of -inf alone); `return_lse` adds the fp32 [rows, q_heads] logsumexp.  Rows of no request are left
    as they were.

    max_width: a bound on the rows of a request, by which the work is laid out (results depend on it
    in the order of their sums alone); default 64 with a tree_mask, else all rows, which costs up to a
    sixth where the requests are many and short (64 requests of 1 row, up to 512 cached, bf16: 81 us
    against 70 with max_width=1).  A tree has at most 64 nodes.
    workspace: uint8 scratch of `workspace_bytes` (allocated for the call unless given); calls that may
    overlap need one each.  err (int32 [1], optional) collects bit 1: a page outside the cache or
    a length past the page table (those positions are unseen, drafted tokens among them; no token
    moves), bit 2: a wait that timed out, whose rows are NaN.  A masked position's K may hold
    anything; V of positions that some row of the request sees reaches the rows that see it alone,
    infinities and NaN included."""
    c = describe(k_cache, v_cache, k_scale, v_scale)
    dev = k_cache.device
    shape = q.shape
    dtype = _DTYPES.get(q.dtype)
    _check(len(shape) == 3 and dtype is not None, "q must be bf16 or fp16 [rows, q_heads, dim]")
    rows, q_heads, dim = shape
    heads = c.heads
    _check(dim == c.dim and dim <= MAX_DIM, "q and the cache must have one dim, at most 128")
    _check(q_heads >= 1 and q_heads % heads == 0 and q_heads <= 4096 * heads,
           "q_heads must be a multiple of the cache's heads, at most 4096 of them each")
    _check(c.dtype == 3 or c.dtype == dtype, "the cache must have q's type or be e4m3")
    _check(page_table.dtype == torch.int32 and page_table.dim() == 2, "page_table must be int32 [requests, pages]")
    batch, pages = page_table.shape
    table_stride, one = page_table.stride()
    _check(one == 1 or pages <= 1, "page_table's rows must be contiguous")
    if batch <= 1:
        table_stride = pages
    _check(table_stride >= pages, "page_table's rows overlap")
    _check(kv_lens.dtype == torch.int32 and kv_lens.shape == (batch,) and kv_lens.is_contiguous(), "kv_lens must be contiguous int32 [requests]")
    page_size = int(page_size)
    _check(page_size >= 1 and c.slots % page_size == 0, "the cache must hold whole pages of page_size slots")
    _check(q.device == dev and page_table.device == dev and kv_lens.device == dev, "tensors must be on one CUDA device")
    if q_indptr is None:
        _check(batch > 0 and rows % batch == 0 or rows == 0, "without q_indptr every request has the same number of rows")
        width = max(1, rows // max(batch, 1))
        _check(tree_mask is None or width <= MAX_NODES, "a draft tree has at most 64 nodes")
        indptr = None
    else:
        _check(q_indptr.dtype == torch.int32 and q_indptr.shape == (batch + 1,) and q_indptr.is_contiguous(),
               "q_indptr must be contiguous int32 [requests + 1]")
        _check(q_indptr.device == dev, "tensors must be on one CUDA device")
        width = (max(rows, 1) if tree_mask is None else MAX_NODES) if max_width is None else int(max_width)
        _check(width >= 1, "max_width must be at least 1")
        indptr = q_indptr.data_ptr()
    mask = None
    if tree_mask is not None:
        _check(tree_mask.dtype == torch.int64 and tree_mask.shape == (rows,) and tree_mask.is_contiguous(),
               "tree_mask must be contiguous int64 [rows]")
        _check(tree_mask.device == dev, "tensors must be on one CUDA device")
        mask = tree_mask.data_ptr()
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    _check(0.0 < scale < 3.4e38, "scale must be positive and finite")
    q_stride, q_head_stride, one = q.stride()
    _check(one == 1 or rows == 0, "rows of q and out must be contiguous")
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=dev)
        out_stride, out_head_stride = q_heads * dim, dim
    else:
        _check(out.shape == shape and out.dtype == q.dtype and out.device == dev, "out must be like q")
        out_stride, out_head_stride, one = out.stride()
        _check(one == 1 or rows == 0, "rows of q and out must be contiguous")
        _check((rows <= 1 or out_stride >= dim) and (q_heads == 1 or out_head_stride >= dim), "the rows of out overlap")
    if lse is not None:
        _check(lse.shape == (rows, q_heads) and lse.dtype == torch.float32 and lse.is_contiguous() and lse.device == dev,
               "lse must be contiguous fp32 [rows, q_heads]")
    elif return_lse:
        lse = torch.empty((rows, q_heads), dtype=torch.float32, device=dev)
    if err is not None:
        check_err(err, dev)
    _check(dev.type == "cuda", "tensors must be on a CUDA device")
    if rows and batch:
        need = workspace_bytes(q_heads, heads, dim, width)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        else:
            _check(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need and workspace.device == dev,
                   "workspace must be workspace_bytes(...) bytes (uint8) on the cache's device")
        if rows == 1:
            q_stride = out_stride = 0
        if q_heads == 1:
            q_head_stride = out_head_stride = 0
        launch("dsv_tree_attention", dev, batch, rows, q_heads, dtype, q.data_ptr(), q_stride, q_head_stride, c,
               page_table.data_ptr() if pages else None, table_stride, pages, page_size, kv_lens.data_ptr(), indptr, width, mask, scale,
               out.data_ptr(), out_stride, out_head_stride, None if lse is None else lse.data_ptr(), None if err is None else err.data_ptr(),
               workspace.data_ptr(), workspace.numel())
    return (out, lse) if return_lse else out
