"""What the KV-cache and draft-tree operators refuse, and the ancestor bits, without a GPU."""

import ctypes

import pytest
import torch

from dspine_b200 import _lib, accept, attention, build, kvcache

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _cache(slots=32, heads=2, dim=64, dtype=torch.bfloat16):
    k, v, ks, vs = kvcache.allocate_kv(slots, heads, dim, dtype=dtype, device="cpu")
    return k, v, ks, vs


def test_tree_mask():
    assert attention.tree_mask(torch.tensor([-1])).tolist() == [1]
    assert attention.tree_mask(torch.tensor([-1, 0, 0, 1, 2, 4])).tolist() == [1, 0b11, 0b101, 0b1011, 0b10101, 0b110101]
    chain = attention.tree_mask(torch.arange(-1, 63))
    assert chain.tolist() == [(1 << (i + 1)) - 1 for i in range(63)] + [-1]
    g = torch.Generator().manual_seed(0)
    parents = torch.tensor([[-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, 64)] for _ in range(5)])
    got = attention.tree_mask(parents)
    for b in range(5):
        masks = []
        for i, p in enumerate(parents[b].tolist()):
            masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        assert [m & (2 ** 64 - 1) for m in got[b].tolist()] == masks
    two_roots = attention.tree_mask(torch.tensor([-1, -1, 1]))
    assert two_roots.tolist() == [1, 2, 6]
    assert attention.tree_mask(torch.zeros(3, 0, dtype=torch.int32)).shape == (3, 0)
    with pytest.raises(ValueError, match="at most 64"):
        attention.tree_mask(torch.zeros(65, dtype=torch.int64))
    with pytest.raises(ValueError, match="integers"):
        attention.tree_mask(torch.zeros(4))


def test_allocate_kv():
    k, v, ks, vs = _cache(dtype=E4M3)
    assert k.dtype is E4M3 and k.shape == (32, 2, 64) and ks.shape == (32, 2) and bool((vs == 1).all())
    k, v, ks, vs = _cache(dtype=torch.float16)
    assert ks is None and not bool(v.any())
    with pytest.raises(ValueError, match="bf16, fp16 or e4m3"):
        kvcache.allocate_kv(4, 1, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="multiple of 16"):
        kvcache.allocate_kv(4, 1, 72, device="cpu")


def test_caches_that_are_refused():
    k, v, ks, vs = _cache(dtype=E4M3)
    at = torch.zeros(3, dtype=torch.int32)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16)

    def refused(match, *, k=rows, v=rows, kc=k, vc=v, slots=at, **more):
        scales = {"k_scale": ks, "v_scale": vs, **more}
        with pytest.raises(ValueError, match=match):
            kvcache.write_kv(k, v, kc, vc, slots, **scales)

    refused("needs k_scale", k_scale=None)
    refused("fp32", k_scale=ks.double())
    refused("fp32", v_scale=vs[:-1])
    refused(r"\[slots, heads, dim\]", kc=k[0], vc=v[0])
    refused(r"\[slots, heads, dim\]", vc=v[:-1])
    refused("bf16, fp16 or e4m3", kc=torch.zeros(32, 2, 64), vc=torch.zeros(32, 2, 64))
    refused("same strides", kc=torch.zeros(32, 2, 128, dtype=torch.uint8).view(E4M3)[:, :, :64])
    refused("multiple of 16", kc=k[:, :, :40], vc=v[:, :, :40])
    refused("not overlap", kc=k[:1].expand(32, 2, 64), vc=v[:1].expand(32, 2, 64))
    refused(r"\[tokens, heads, dim\]", k=rows[:, :1], v=rows[:, :1])
    refused("bf16, fp16 or fp32", k=rows.double(), v=rows.double())
    refused("rows must be contiguous", k=torch.zeros(3, 64, 2, dtype=torch.bfloat16).transpose(1, 2))
    refused("slots must be", slots=at[:2])
    refused("int32 or int64", slots=at.float())
    refused("contiguous", slots=torch.zeros(6, dtype=torch.int32)[::2])
    refused("err must be", err=torch.zeros(2, dtype=torch.int32))
    refused("CUDA device")                                 # all else is right
    b, c, _, _ = _cache()
    with pytest.raises(ValueError, match="rows of its own type"):
        kvcache.write_kv(rows.half(), rows.half(), b, c, at)
    with pytest.raises(ValueError, match="only an e4m3 cache"):
        kvcache.write_kv(rows, rows, b, c, at, k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="read as"):
        kvcache.read_kv(b, c, at, dtype=torch.int32)
    with pytest.raises(ValueError, match="out must be"):
        kvcache.read_kv(b, c, at, out=(rows, rows[:2]))
    with pytest.raises(ValueError, match="CUDA device"):
        kvcache.read_kv(b, c, at)


def test_attention_refusals():
    k, v, _, _ = _cache()
    q = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    starts = torch.tensor([0, 3, 6], dtype=torch.int32)
    good = dict(q=q, k_cache=k, v_cache=v, page_table=table, kv_lens=lens, page_size=8, q_indptr=starts,
                tree_mask=torch.zeros(6, dtype=torch.int64))

    def refused(match, **more):
        with pytest.raises(ValueError, match=match):
            attention.tree_attention(**{**good, **more})

    refused("CUDA device")                                 # all else is right
    refused("bf16 or fp16", q=q.float())
    refused("q's type or be e4m3", q=q.half())
    refused("one dim", q=q[:, :, :32])
    refused("multiple of the cache's heads", q=q[:, :3])
    refused("page_table must be int32", page_table=table.long())
    refused("page_table's rows must be contiguous", page_table=torch.zeros(4, 2, dtype=torch.int32).t())
    refused("page_table's rows overlap", page_table=table[:1].expand(2, 4))
    refused("kv_lens", kv_lens=lens[:1])
    refused("kv_lens", kv_lens=lens.long())
    refused("whole pages", page_size=5)
    refused("whole pages", page_size=0)
    refused("q_indptr must be", q_indptr=starts.long())
    refused("q_indptr must be", q_indptr=starts[:2])
    refused("max_width", max_width=0)
    refused("tree_mask must be", tree_mask=torch.zeros(5, dtype=torch.int64))
    refused("tree_mask must be", tree_mask=torch.zeros(6, dtype=torch.int32))
    refused("at most 64 nodes", q_indptr=None, q=torch.zeros(130, 4, 64, dtype=torch.bfloat16), tree_mask=torch.zeros(130, dtype=torch.int64))
    refused("same number of rows", q_indptr=None, q=q[:5], tree_mask=None)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused("scale must be", scale=scale)
    refused("out must be like q", out=q.half())
    refused("rows of out overlap", out=q[:1].expand(6, 4, 64))
    refused("must be contiguous", q=torch.zeros(6, 64, 4, dtype=torch.bfloat16).transpose(1, 2))
    refused("lse must be", lse=torch.zeros(6, 3))
    refused("err must be", err=torch.zeros(1))
    wide, wide_v, _, _ = _cache(dim=144)
    refused("at most 128", q=torch.zeros(6, 4, 144, dtype=torch.bfloat16), k_cache=wide, v_cache=wide_v)


def test_accept_tree_refusals():
    t = torch.zeros(2, 8, dtype=torch.int64)
    good = dict(tokens=t, top1=t, tree_mask=t)

    def refused(match, **more):
        with pytest.raises(ValueError, match=match):
            accept.accept_tree(**{**good, **more})

    refused("CUDA device")
    refused("top1 must be", top1=t[:1])
    refused("tree_mask must be", tree_mask=t.int())
    refused("tokens must be contiguous", tokens=torch.zeros(8, 2, dtype=torch.int64).t())
    refused(r"tokens must be \[requests, nodes\]", tokens=t.view(-1))
    refused("hold every node", width=7)
    refused("at most 64", width=65)
    refused("at most 64", tokens=torch.zeros(1, 65, dtype=torch.int64))
    refused(r"tokens must be \[rows\]", q_indptr=torch.zeros(3, dtype=torch.int32))
    flat = dict(tokens=t.view(-1), top1=t.view(-1), tree_mask=t.view(-1))
    refused("q_indptr must be", **flat, q_indptr=torch.zeros(3, dtype=torch.int64))
    refused("q_indptr must be", **flat, q_indptr=torch.zeros(0, dtype=torch.int32))
    refused("prefix_lens", prefix_lens=torch.zeros(3, dtype=torch.int32))
    refused("slots must be", slots=t)
    refused("outputs must be", outputs=accept.TreeAccept.allocate(2, 9, "cpu"))
    refused("outputs must be", slots=t.int(), outputs=accept.TreeAccept.allocate(2, 8, "cpu", slots=False))


def test_c_entries_refuse_before_launch(lib):
    def cache(**more):
        c = dict(k=16, v=16, k_scale=16, v_scale=16, slots=64, slot_stride=128, head_stride=64, scale_stride=2, heads=2,
                 dim=64, dtype=0)
        return _lib.KvCache(**{**c, **more})

    def write(c, n=1, dtype=0, k=16, ks=128, kh=64, slots=16, s64=0, err=None):
        return lib.dsv_kv_write(n, dtype, k, ks, kh, 16, 128, 64, slots, s64, c, err, None)

    assert write(cache(), n=0) == 0 and write(cache(), n=-1) == 1
    assert write(None) == 3 and write(cache(k=None)) == 3 and write(cache(), slots=None) == 3 and write(cache(), k=None) == 3
    assert write(cache(dtype=1)) == 2 and write(cache(), dtype=3) == 2 and write(cache(), dtype=2) == 2
    assert write(cache(dtype=3, v_scale=None, slot_stride=128)) == 3
    for bad in (dict(slots=0), dict(slots=1 << 31), dict(heads=0), dict(dim=24), dict(dim=272), dict(head_stride=48), dict(slot_stride=48)):
        assert write(cache(**bad)) == 1, bad
    assert write(cache(dtype=3, scale_stride=1)) == 1
    assert write(cache(), n=1 << 30) == 1                  # tokens * heads past 2^31
    assert write(cache(k=8)) == 4 and write(cache(slot_stride=132)) == 4 and write(cache(dtype=3, head_stride=72)) == 4
    assert write(cache(), ks=130) == 4 and write(cache(), k=24) == 4 and write(cache(), slots=18) == 4
    assert write(cache(), slots=20, s64=1) == 4 and write(cache(), err=18) == 4

    def read(c, n=1, dtype=0, out=16, slots=16):
        return lib.dsv_kv_read(n, slots, 0, c, dtype, out, 16, None, None)

    assert read(cache(), n=0) == 0 and read(cache(), n=-1) == 1 and read(cache(), dtype=3) == 2
    assert read(cache(), out=None) == 3 and read(cache(), out=8) == 4 and read(cache(), slots=None) == 3

    size = ctypes.c_size_t()
    ws = lib.dsv_tree_attention_workspace_size
    assert ws(8, 2, 64, 16, ctypes.byref(size)) == 0 and ws(8, 2, 64, 16, None) == 3
    for bad in ((8, 0, 64, 1), (7, 2, 64, 1), (8, 2, 72, 1), (8, 2, 144, 1), (8, 2, 64, 0)):
        assert ws(*bad, ctypes.byref(size)) == 1

    def attend(c=None, batch=2, rows=6, heads=4, dtype=0, q=16, qs=256, table=16, ts=4, pages=4, page=8, lens=16, ind=16,
               width=3, mask=None, scale=0.1, out=16, lse=None, err=None, wsp=16, nbytes=1 << 40):
        return lib.dsv_tree_attention(batch, rows, heads, dtype, q, qs, 64, c or cache(), table, ts, pages, page, lens, ind,
                                      width, mask, scale, out, 256, 64, lse, err, wsp, nbytes, None)

    assert attend(batch=0, rows=0) == 0 and attend(rows=0) == 0
    assert attend(dtype=1) == 2 and attend(dtype=2) == 2 and attend(cache(dtype=1)) == 2
    for bad in (dict(batch=-1), dict(rows=-1), dict(heads=5), dict(heads=0), dict(page=0), dict(page=5), dict(pages=-1),
                dict(ts=3), dict(width=0), dict(pages=1 << 29, ts=1 << 29), dict(ind=None, rows=7),
                dict(ind=None, rows=130, width=65, mask=16)):
        assert attend(**bad) == 1, bad
    assert attend(cache(dim=144, head_stride=144, slot_stride=288)) == 1
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert attend(scale=scale) == 8
    for bad in (dict(q=None), dict(out=None), dict(lens=None), dict(table=None)):
        assert attend(**bad) == 3, bad
    for bad in (dict(q=8), dict(qs=260), dict(out=24), dict(table=18), dict(lens=18), dict(ind=18), dict(mask=12), dict(lse=18),
                dict(err=18)):
        assert attend(**bad) == 4, bad
    if lib.dsv_tree_attention_workspace_size(4, 2, 64, 3, ctypes.byref(size)) == 0 and size.value:
        assert attend(nbytes=size.value - 1) == 6 and attend(wsp=None) == 3 and attend(wsp=8) == 4

    def tree(batch=2, rows=6, ind=16, nodes=3, width=8, tokens=16, kept=16, slots=16, out=16):
        return lib.dsv_accept_tree(batch, rows, tokens, 16, 16, ind, nodes, None, slots, width, 16, 16, 16, out, 16, kept, 16, None)

    assert tree(batch=0, rows=0) == 0
    for bad in (dict(batch=-1), dict(rows=-1), dict(width=0), dict(width=65), dict(ind=None, rows=7), dict(ind=None, nodes=9, rows=18)):
        assert tree(**bad) == 1, bad
    assert tree(tokens=None) == 3 and tree(slots=None) == 3 and tree(out=None) == 3
    assert tree(tokens=12) == 4 and tree(out=12) == 4 and tree(ind=18) == 4


def test_positions_near_the_end_of_32_bits_are_refused(lib):
    """A tile past the last position would not be told from one at its start."""
    c = _lib.KvCache(k=16, v=16, k_scale=None, v_scale=None, slots=64, slot_stride=128, head_stride=64, scale_stride=2, heads=2,
                     dim=64, dtype=0)

    def attend(pages, page):
        return lib.dsv_tree_attention(1, 1, 4, 0, 16, 256, 64, c, 16, pages, pages, page, 16, 16, 1, None, 0.1, 16, 256, 64, None,
                                      None, 16, 0, None)

    assert attend((1 << 27) - 1, 16) == 1 and attend((1 << 31) - 1, 1) == 1
    assert attend((1 << 27) - 16, 16) == 6                  # the positions are taken: the workspace is too small


def test_rows_of_queries_past_32_bits_are_refused(lib):
    c = _lib.KvCache(k=16, v=16, k_scale=None, v_scale=None, slots=64, slot_stride=16, head_stride=16, scale_stride=1, heads=1,
                     dim=16, dtype=0)

    def attend(rows, heads):
        return lib.dsv_tree_attention(1, rows, heads, 0, 16, 16, 16, c, 16, 4, 4, 16, 16, 16, 1, None, 0.1, 16, 16, 16, None, None,
                                      16, 0, None)

    assert attend(1 << 30, 2) == 1 and attend((1 << 31) - 1, 1) == 1 and attend(1 << 20, 4096) == 1
    assert attend((1 << 30) - 128, 2) == 6                  # taken: the workspace is too small


def test_limits_of_waits_that_are_refused(lib):
    for bad in ((0, -1), (-1, -1), (2000001, -1), (1000, -2)):
        assert lib.dsv_tree_attention_waits(*bad) == 1
    assert lib.dsv_tree_attention_waits(2000000, -1) == 0


@pytest.mark.parametrize("name", ["accept", "commit", "bonus", "output", "path", "kept", "new_seq"])
def test_every_output_of_accept_tree_has_to_be_aligned(lib, name):
    size = {"bonus": 8, "output": 8}.get(name, 4)
    out = dict(accept=16, commit=16, bonus=16, output=16, path=16, kept=16, new_seq=16)

    def tree(**more):
        o = {**out, **more}
        return lib.dsv_accept_tree(1, 3, 16, 16, 16, 16, 3, None, 16, 8, o["accept"], o["commit"], o["bonus"], o["output"], o["path"],
                                   o["kept"], o["new_seq"], None)

    for off in range(1, size):
        assert tree(**{name: 16 + off}) == 4, off


def test_sizes_of_workspaces_are_not_kept_for_every_width(lib):
    """A server asks with another width at nearly every step."""
    for width in list(range(1, 2000)) + [1, 5, 1999]:
        size = ctypes.c_size_t()
        assert lib.dsv_tree_attention_workspace_size(32, 8, 128, width, ctypes.byref(size)) == 0
        assert attention.workspace_bytes(32, 8, 128, width) == size.value
    assert attention.workspace_bytes.cache_info().currsize <= 64
