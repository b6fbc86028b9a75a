"""Waits of tree_attention that run out: tiles that are never announced, under a limit of 20 ms."""

import pytest
import torch

from test_gpu_tree_attention import Case

from dspine_b200 import _lib, attention

pytestmark = pytest.mark.gpu


@pytest.fixture
def held():
    yield lambda tile: _lib.call("dsv_tree_attention_waits", 20000, tile)
    _lib.call("dsv_tree_attention_waits", 2000000, -1)


@pytest.mark.parametrize("kind,cache,dim", [("bf16", "bf16", 128), ("bf16", "e4m3", 128), ("fp16", "e4m3", 64), ("fp16", "fp16", 64)])
@pytest.mark.parametrize("tile", [0, 1, 17, 34])      # a block has 34 or 35 tiles
def test_rows_whose_tiles_never_come_are_nan(held, kind, cache, dim, tile):
    """No row passes for a result: those of a block that gave up are NaN in out and lse, the others right, the word
    says so, and the next call is as if nothing had been."""
    c = Case([1, 16, 40, 3, 64] * 4, [30, 700, 90, 9000, 200] * 4, heads=32, kv_heads=8, dim=dim, page=16, kind=kind, cache=cache, tree=True,
             seed=1)
    a, k = c.args()
    good, good_lse = attention.tree_attention(*a, **k)
    held(tile)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = torch.full_like(good, 5.0), torch.full_like(good_lse, 5.0)
    attention.tree_attention(*a, **{**k, "out": out, "lse": lse, "err": err})
    assert int(err) == 4
    gone = torch.isnan(lse)
    assert bool(gone.any()) and bool(gone.all()) == (tile < 34)
    assert torch.equal(torch.isnan(out), gone[..., None].expand_as(out))
    assert torch.equal(out[~gone], good[~gone]) and torch.equal(lse[~gone], good_lse[~gone])
    plain = attention.tree_attention(*a, **k)[1]           # without a word to tell it in
    assert torch.equal(torch.isnan(plain), gone)
    _lib.call("dsv_tree_attention_waits", 2000000, -1)
    again, again_lse = attention.tree_attention(*a, **{**k, "err": err.zero_()})
    assert int(err) == 0 and torch.equal(again, good) and torch.equal(again_lse, good_lse)


def test_a_short_context_in_one_tile(held):
    """Items of one tile are never joined: their rows are NaN all the same."""
    c = Case([1, 2], [30, 64], heads=8, kv_heads=2, dim=64, page=64, seed=2)
    a, k = c.args()
    k["out"] = torch.full_like(a[0], 5.0)
    held(0)
    out, lse = attention.tree_attention(a[0], a[1], a[2], a[3][:, :1].contiguous(), a[4], **k)
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())
