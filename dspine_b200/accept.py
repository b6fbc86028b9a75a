"""Host API of the per-request accept steps (C ABI: dsv_accept_greedy, dsv_accept_compact,
dsv_accept_tree).

`accept_greedy` is verification/caps.py:32-59 `_accept_capped` on the GPU: the five accept
outputs of a greedy (argmax) verification from the target's top-1 ids.  `accept_compact`
packs accepted tokens and KV slots after any accept step (SGLang's `_commit_accept`, wrapped
at runtime/worker.py:745-777).  `accept_tree` is the greedy accept for draft trees.  Argument errors raise ValueError before launch.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from .kvcache import launch
from .verify import CompactOutputs, Workspace, new_outputs, workspace_for  # noqa: F401

T = 16


def _check(cond, msg):
    if not cond:
        raise ValueError(msg)


def _stream(device) -> int:
    return torch.cuda.current_stream(torch.device(device)).cuda_stream


def accept_greedy(candidates, top1, verify_lens, prefix_lens=None, *, outputs=None):
    """candidates [B,16] int64; top1 [B,16] int64 (any stride along the last dim, e.g. column 0
    of a [B*16, k] top-k id array viewed as [B,16]); verify_lens [B] int32; prefix_lens [B]
    int32 (zeros when None).  Returns (accept, commit, bonus, output, new_seq)."""
    _check(candidates.dim() == 2 and candidates.shape[1] == T and candidates.dtype == torch.int64
           and candidates.is_contiguous(), "candidates must be contiguous int64 [B,16]")
    B = candidates.shape[0]
    dev = candidates.device
    _check(top1.shape == (B, T) and top1.dtype == torch.int64 and top1.device == dev,
           "top1 must be int64 [B,16]")
    s = top1.stride(1)
    _check(s >= 1 and top1.stride(0) == T * s, "top1 must be a uniformly strided [B,16] view")
    _check(verify_lens.shape == (B,) and verify_lens.dtype == torch.int32, "verify_lens int32 [B]")
    if prefix_lens is None:
        prefix_lens = torch.zeros(B, dtype=torch.int32, device=dev)
    _check(prefix_lens.shape == (B,) and prefix_lens.dtype == torch.int32, "prefix_lens int32 [B]")
    if outputs is None:
        outputs = new_outputs(B, dev)
    _lib.call("dsv_accept_greedy", B, candidates.data_ptr(), top1.data_ptr(), s,
              verify_lens.contiguous().data_ptr(), prefix_lens.contiguous().data_ptr(),
              *(o.data_ptr() for o in outputs), _stream(dev))
    return outputs


def accept_compact(commit, verify_lens, output, slots, slot_rows, *, compact=None,
                   workspace: Workspace | None = None):
    """Pack output[b, :commit_b] and the KV slots of positions [0, commit_b) of every request
    (and the freed slots of positions [commit_b, verify_len_b)) by the exclusive scan of commit."""
    B = commit.shape[0]
    dev = commit.device
    _check(commit.dtype == torch.int32 and verify_lens.dtype == torch.int32, "int32 commit/lens")
    _check(output.shape == (B, T) and output.dtype == torch.int64, "output int64 [B,16]")
    _check(slots.dtype == torch.int32 and slot_rows.dtype == torch.int64 and slot_rows.shape == (B,),
           "slots int32, slot_rows int64 [B]")
    if compact is None:
        compact = CompactOutputs.allocate(B, dev)
    if workspace is None:
        workspace = workspace_for(B, dev)
    c = _lib.CompactOut(slots.data_ptr(), slots.numel(), slot_rows.data_ptr(),
                        compact.tokens.data_ptr(), compact.kept_slots.data_ptr(),
                        compact.offsets.data_ptr(), compact.freed_slots.data_ptr(),
                        compact.freed_offsets.data_ptr())
    _lib.call("dsv_accept_compact", B, commit.data_ptr(), verify_lens.data_ptr(),
              output.contiguous().data_ptr(), ctypes.byref(c), workspace.buf.data_ptr(),
              _stream(dev))
    return compact


@dataclass
class TreeAccept:
    """Outputs of accept_tree (see there)."""

    accept: torch.Tensor
    commit: torch.Tensor
    bonus: torch.Tensor
    output: torch.Tensor
    path: torch.Tensor
    kept_slots: torch.Tensor | None
    new_seq: torch.Tensor

    @staticmethod
    def allocate(batch: int, width: int, device, *, slots=True) -> "TreeAccept":
        """Outputs for `batch` requests."""
        accept, commit, new_seq = torch.empty((3, batch), dtype=torch.int32, device=device).unbind()
        path, *kept = torch.empty((2 if slots else 1, batch, width), dtype=torch.int32, device=device).unbind()
        return TreeAccept(accept, commit, torch.empty(batch, dtype=torch.int64, device=device),
                          torch.empty((batch, width), dtype=torch.int64, device=device), path, kept[0] if slots else None, new_seq)

    def _check(self, batch, width, dev, slots):
        for x, shape, dtype in ((self.accept, (batch,), torch.int32), (self.commit, (batch,), torch.int32), (self.bonus, (batch,), torch.int64),
                                (self.output, (batch, width), torch.int64), (self.path, (batch, width), torch.int32),
                                (self.new_seq, (batch,), torch.int32)) + (((self.kept_slots, (batch, width), torch.int32),) if slots else ()):
            _check(x is not None and x.shape == shape and x.dtype == dtype and x.device == dev and x.is_contiguous(),
                   "outputs must be as TreeAccept.allocate gives them")


def accept_tree(tokens, top1, tree_mask, *, q_indptr=None, prefix_lens=None, slots=None, width=None, outputs=None):
    """Greedy acceptance over draft trees (C ABI: dsv_accept_tree), the tree form of accept_greedy.

    tokens, top1, tree_mask [rows] int64: each drafted node's token, the target's top-1 token at
    it and its ancestor bits (`attention.tree_mask`); node 0 of a request is the root, its last
    committed token.  Request b owns rows [q_indptr[b], q_indptr[b+1]) (int32 [B+1]; None: tokens
    is [B, nodes], and so are top1, tree_mask and slots).  A node is accepted when its token and those of all its ancestors are
    the top-1 token of their parent; the deepest accepted node, the first among equals, ends the
    path.  Returns TreeAccept: accept [B] (drafted nodes on the path), commit = accept + 1, bonus
    [B] int64 (the top-1 token after the path), output [B, width] int64 (the path's tokens after
    the root, the bonus, then 0), path [B, width] int32 (its nodes, then -1), kept_slots [B,
    width] int32 (slots of its nodes, then -1; None without slots), new_seq = prefix_lens (zeros
    when None) + commit.  At most the first `width` (<= 64, default 64 or nodes) rows of a request
    are looked at; a request without rows gets commit 0 and bonus -1."""
    dev = tokens.device
    shape = tokens.shape
    if q_indptr is None:
        _check(len(shape) == 2, "without q_indptr tokens must be [requests, nodes]")
        B, nodes = shape
        width = max(1, nodes) if width is None else int(width)
        _check(nodes <= width, "width must hold every node")
        indptr, rows = None, B * nodes
    else:
        _check(len(shape) == 1, "with q_indptr tokens must be [rows]")
        _check(q_indptr.dim() == 1 and q_indptr.shape[0] >= 1 and q_indptr.dtype == torch.int32 and q_indptr.device == dev
               and q_indptr.is_contiguous(), "q_indptr must be contiguous int32 [requests + 1]")
        B, nodes = q_indptr.shape[0] - 1, 0
        width = 64 if width is None else int(width)
        indptr, rows = q_indptr.data_ptr(), shape[0]
    _check(1 <= width <= 64, "a draft tree has at most 64 nodes")
    for x in (tokens, top1, tree_mask):
        if x.dtype != torch.int64 or x.shape != shape or x.device != dev or not x.is_contiguous():
            name = "tokens" if x is tokens else ("top1" if x is top1 else "tree_mask")
            _check(False, f"{name} must be contiguous int64, one value a node")
    if prefix_lens is not None:
        _check(prefix_lens.dtype == torch.int32 and prefix_lens.shape == (B,) and prefix_lens.device == dev and prefix_lens.is_contiguous(),
               "prefix_lens must be contiguous int32 [requests]")
    if slots is not None:
        _check(slots.dtype == torch.int32 and slots.shape == shape and slots.device == dev and slots.is_contiguous(),
               "slots must be contiguous int32, one value a node")
    if outputs is None:
        outputs = TreeAccept.allocate(B, width, dev, slots=slots is not None)
    else:
        outputs._check(B, width, dev, slots is not None)
    _check(dev.type == "cuda", "tensors must be on a CUDA device")
    o = outputs
    if B:
        launch("dsv_accept_tree", dev, B, rows, tokens.data_ptr(), top1.data_ptr(), tree_mask.data_ptr(), indptr, nodes,
               None if prefix_lens is None else prefix_lens.data_ptr(), None if slots is None else slots.data_ptr(), width,
               o.accept.data_ptr(), o.commit.data_ptr(), o.bonus.data_ptr(), o.output.data_ptr(), o.path.data_ptr(),
               None if slots is None else o.kept_slots.data_ptr(), o.new_seq.data_ptr())
    return outputs
