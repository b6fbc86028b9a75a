"""tree_attention on the GPU against 64-bit attention, row by row over the keys that each row sees."""

import math

import pytest
import torch

import kv_reference as R

from dspine_b200 import accept, attention, kvcache

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": R.E4M3}


def _parents(g, n):
    return [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, n)]


class Case:
    """One batch: queries, a cache whose unused slots hold NaN, shuffled pages, lengths, masks."""

    def __init__(self, widths, lengths, *, heads=8, kv_heads=2, dim=64, page=16, kind="bf16", cache="bf16", tree=False,
                 seed=0, tail=0, size=1.0):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page, self.group, self.kind, self.cache = g, page, heads // kv_heads, TYPES[kind], cache
        self.widths, self.lengths = widths, lengths
        self.starts = [0]
        for w in widths:
            self.starts.append(self.starts[-1] + w)
        rows = self.starts[-1] + tail
        self.q = (size * torch.randn(rows, heads, dim, generator=g)).to(self.kind)
        pages = [-(-n // page) for n in lengths]
        self.pages = sum(pages) + 2
        order = torch.randperm(self.pages, generator=g).int()
        self.table = torch.full((len(widths), max(pages + [1]) + 1), 1 << 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = order[at:at + n]
            at += n
        slots = self.pages * page
        k, v = torch.randn(slots, kv_heads, dim, generator=g), torch.randn(slots, kv_heads, dim, generator=g) + 0.3
        used = torch.zeros(slots, dtype=torch.bool)
        for b, n in enumerate(lengths):
            pos = torch.arange(n)
            used[self.table[b][pos // page].long() * page + pos % page] = True
        self.ks = self.vs = None
        if cache == "e4m3":
            v = v * torch.exp(2 * torch.randn(slots, kv_heads, 1, generator=g))    # scales far apart
            (self.k, self.ks), (self.v, self.vs) = R.quantise(k), R.quantise(v)
            for c, s in ((self.k, self.ks), (self.v, self.vs)):
                c.view(torch.uint8)[~used] = 0x7F
                s[~used] = math.nan
        else:
            self.k, self.v = k.to(TYPES[cache]), v.to(TYPES[cache])
            self.k[~used], self.v[~used] = math.nan, math.inf
        self.masks = None
        if tree:
            self.masks = torch.cat([attention.tree_mask(torch.tensor(_parents(g, w))) if w else torch.zeros(0, dtype=torch.int64)
                                    for w in widths] + [torch.zeros(tail, dtype=torch.int64)])
        self.scale = 1.0 / math.sqrt(dim)

    def args(self):
        d = lambda x: None if x is None else x.cuda()  # noqa: E731
        return (d(self.q), d(self.k), d(self.v), d(self.table), torch.tensor(self.lengths, dtype=torch.int32).cuda()), dict(
            page_size=self.page, q_indptr=torch.tensor(self.starts, dtype=torch.int32).cuda(), tree_mask=d(self.masks),
            scale=self.scale, k_scale=d(self.ks), v_scale=d(self.vs), return_lse=True)

    def want(self):
        return R.attention(self.q, R.cache_values(self.k, self.ks), R.cache_values(self.v, self.vs), self.table, self.lengths,
                           page_size=self.page, starts=self.starts, masks=self.masks, scale=self.scale, group=self.group,
                           pages=self.pages)

    def check(self, got, want=None):
        out, lse = (x.double().cpu() for x in got)
        want = want or self.want()
        n = self.starts[-1]
        # weights are rounded to the operand type: fp16 for an e4m3 cache, else the cache's own
        half = R.HALF_STEP[torch.float16 if self.cache == "e4m3" else self.kind]
        bound, lse_bound = R.attention_bounds(*want, dim=self.q.shape[2], out_dtype=self.kind, weight_half_step=half)
        w_out, w_lse = want[0][:n], want[1][:n]
        fine = torch.isfinite(w_out)
        off = (out[:n] - w_out).abs()
        assert torch.equal(torch.isfinite(out[:n]), fine)
        assert bool((off[fine] <= bound[:n][fine]).all()), (float((off[fine] / bound[:n][fine]).max()), "times the bound")
        assert torch.equal(out[:n][~fine].nan_to_num(1.0, 2.0, 3.0), w_out[~fine].nan_to_num(1.0, 2.0, 3.0))
        empty = torch.isneginf(w_lse)
        assert torch.equal(torch.isneginf(lse[:n]), empty)
        ok = torch.isfinite(w_lse)
        assert bool(((lse[:n] - w_lse).abs()[ok] <= lse_bound[:n][ok]).all())

    def run(self, **more):
        a, k = self.args()
        return attention.tree_attention(*a, **{**k, **more})


GRID = [
    dict(widths=[1], lengths=[1]),
    dict(widths=[1], lengths=[333], heads=32, kv_heads=8, dim=128),
    dict(widths=[1, 1, 1], lengths=[127, 128, 129], dim=128),
    dict(widths=[1] * 5, lengths=[1, 2, 700, 64, 65], heads=7, kv_heads=1, dim=80, page=1),
    dict(widths=[16, 3, 9], lengths=[16, 500, 137], heads=32, kv_heads=8, dim=128, page=1),
    dict(widths=[64, 33], lengths=[400, 64], heads=16, kv_heads=2, dim=128, page=64),
    dict(widths=[13, 0, 1, 5], lengths=[300, 40, 1, 1021], heads=14, kv_heads=2, dim=64, page=8),
    dict(widths=[2, 2], lengths=[1000, 3], heads=40, kv_heads=2, dim=96, page=3),
    dict(widths=[4], lengths=[2500], heads=3, kv_heads=3, dim=112, page=7),
    dict(widths=[6, 1], lengths=[257, 1], heads=64, kv_heads=1, dim=16, page=16),
    dict(widths=[10], lengths=[60], heads=48, kv_heads=4, dim=48, page=5),
    dict(widths=[1], lengths=[4099], heads=130, kv_heads=1, dim=32, page=16),
]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("i", range(len(GRID)))
def test_against_64_bits(i, kind, cache, tree):
    c = Case(**GRID[i], kind=kind, cache=cache, tree=tree, seed=i)
    c.check(c.run())


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("width,length", [(65, 65), (100, 300), (257, 257), (200, 1500)])
def test_long_chains(width, length, cache):
    """Without a tree a request may have any number of rows: a chunk of a prompt, causal."""
    c = Case([width, 1, 70], [length, 50, 90], heads=8, kv_heads=2, dim=128, page=16, cache=cache, seed=3)
    c.check(c.run())


@pytest.mark.parametrize("most,tree", [(3, False), (64, True)])
@pytest.mark.parametrize("cache,page", [("bf16", 16), ("e4m3", 1)])
def test_many_short_segments(cache, page, most, tree):
    """More requests than CTAs have room for at once: every CTA goes from segment to segment, and every
    wait of every call has to end."""
    g = torch.Generator().manual_seed(most)
    widths = torch.randint(0, most + 1, (90,), generator=g).tolist()
    lengths = [w + int(n) for w, n in zip(widths, torch.randint(0, 200, (90,), generator=g))]
    c = Case(widths, lengths, heads=32, kv_heads=8, dim=128, page=page, cache=cache, tree=tree, seed=most)
    want, err = c.want(), torch.zeros(1, dtype=torch.int32, device="cuda")
    a, k = c.args()
    for _ in range(20):
        got = attention.tree_attention(*a, **k, max_width=most, err=err)
    assert int(err) == 0
    c.check(got, want)


@pytest.mark.parametrize("tree", [False, True])
def test_more_requests_than_threads(tree):
    """1100 requests, some without rows, some with fewer cached positions than rows."""
    g = torch.Generator().manual_seed(5)
    widths = torch.randint(0, 4, (1100,), generator=g).tolist()
    lengths = torch.randint(0, 150, (1100,), generator=g).tolist()
    lengths[7], widths[7], lengths[8], widths[8] = 0, 3, 2, 3
    c = Case(widths, lengths, heads=2, kv_heads=2, dim=16, page=4, tree=tree, seed=5)
    c.check(c.run())


def test_the_layout_bound_does_not_change_what_is_computed():
    c = Case([40, 2, 17], [300, 700, 17], heads=16, kv_heads=2, dim=64, seed=4)
    want = c.want()
    for w in (1, 16, 40, 64, 1000):
        c.check(c.run(max_width=w), want)


def test_equal_widths_without_offsets():
    c = Case([5] * 4, [9, 5, 300, 130], heads=8, kv_heads=4, dim=64, tree=True, seed=5)
    c.check(c.run(q_indptr=None))


def test_rows_that_see_nothing():
    """Masks of zeros on an empty context, lengths of zero, drafted tokens that were never cached."""
    c = Case([3, 2, 4, 1], [3, 0, 2, 200], tree=True, seed=6)
    c.masks[0] = 0
    c.masks[2] = 0b100
    out, lse = got = c.run()
    c.check(got)
    assert not bool(out[0].any()) and bool(torch.isneginf(lse[0]).all())
    assert not bool(out[3:5].any()) and bool(torch.isneginf(lse[3:5]).all())
    c.masks = None
    out, lse = got = c.run()              # request 2: 4 rows, 2 cached positions, so rows 0 and 1 see none
    c.check(got)
    assert not bool(out[5:7].any()) and bool(torch.isneginf(lse[5:7]).all()) and bool(out[7].any())


@pytest.mark.parametrize("bits", [-1, -(1 << 63), 0])
def test_extreme_masks(bits):
    """All bits, the sign bit alone, none: bits past the drafted tokens are not seen."""
    c = Case([64, 5, 63], [64, 100, 300], tree=True, seed=7)
    c.masks[:] = bits
    c.check(c.run())


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_masked_infinities_and_nan_do_not_reach_a_row(cache):
    """A drafted token whose K or V is NaN or infinite reaches only the rows that see it."""
    c = Case([6, 40], [150, 60], heads=16, kv_heads=2, dim=64, page=16, cache=cache, tree=True, seed=8)
    c.masks[:6] = torch.tensor([0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100001])

    def slot(b, pos):
        return int(c.table[b, pos // 16]) * 16 + pos % 16

    for b, j, what in ((0, 2, "v"), (0, 3, "k"), (1, 39, "v"), (1, 38, "k")):
        at = slot(b, c.lengths[b] - c.widths[b] + j)
        if cache == "e4m3":
            (c.v if what == "v" else c.k).view(torch.uint8)[at, 0, 5] = 0xFF
        else:
            (c.v if what == "v" else c.k)[at, 0, 5] = -math.inf if what == "v" else math.nan
    c.masks[6:] &= (1 << 38) - 1
    c.masks[6 + 38] = (1 << 38) | 1
    c.masks[6 + 39] = (1 << 39) | 1
    out, lse = got = c.run()
    want = c.want()
    n = 46
    nan_rows = torch.isnan(want[1][:n])
    assert torch.equal(torch.isnan(lse.cpu()), nan_rows)                 # a NaN score is a NaN sum
    clean = torch.isfinite(want[0][:n])
    assert torch.equal(torch.isfinite(out.cpu()), clean)
    bound, lse_bound = R.attention_bounds(*want, dim=64, out_dtype=torch.bfloat16, weight_half_step=2.0 ** -8)
    off = (out.double().cpu() - want[0][:n]).abs()
    assert bool((off[clean] <= bound[:n][clean]).all())
    inf = torch.isinf(want[0][:n])
    assert torch.equal(out.double().cpu()[inf], want[0][:n][inf])


def test_nan_in_the_context_reaches_every_row_of_its_head():
    c = Case([4], [300], heads=4, kv_heads=2, dim=64, seed=9)
    c.v[int(c.table[0, 3]) * 16 + 2, 1, 7] = math.nan
    out, _ = c.run()
    bad = torch.isnan(out)
    assert bool(bad[:, 2:, 7].all()) and int(bad.sum()) == 8


def test_large_scores_and_scales():
    """Scores in the hundreds, where a few keys carry the whole weight; scale 1 and a tiny one."""
    for scale in (1.0, 1e-3, 40.0):
        c = Case([4, 9], [500, 130], heads=8, kv_heads=2, dim=128, kind="fp16", cache="fp16", seed=10)
        c.scale = scale
        c.check(c.run())
        c = Case([4, 9], [500, 130], heads=8, kv_heads=2, dim=128, cache="e4m3", seed=11, size=30.0)
        c.scale = scale
        c.check(c.run())


def test_a_rising_maximum():
    """Every next key scores higher than the last: the running maximum moves at each step."""
    c = Case([2], [1500], heads=4, kv_heads=1, dim=64, seed=12)
    c.q[:] = 0
    c.q[..., 0] = 4.0
    pos = torch.arange(1500)
    at = c.table[0][pos // 16].long() * 16 + pos % 16
    c.k[at, 0, 0] = (pos.float() * 0.4).bfloat16()
    c.check(c.run())
    c.k[at, 0, 0] = (-pos.float() * 0.4).bfloat16()
    c.check(c.run())


def test_a_sink_before_many_small_weights():
    """One key of half the weight before thousands that share the rest: small weights keep their sum."""
    for cache in ("bf16", "e4m3"):
        c = Case([1], [6000], heads=2, kv_heads=1, dim=64, seed=13)
        pos = torch.arange(6000)
        at = c.table[0][pos // 16].long() * 16 + pos % 16
        c.q[:] = 0
        c.q[..., 0] = 8.0
        k, v = torch.zeros(c.k.shape), torch.zeros(c.v.shape)
        k[at[0], 0, 0] = math.log(5999.0)                 # scale 1/8: its score is log(5999), the others' 0
        v[at] = 1.0
        v[at[0]] = -1.0
        c.cache = cache
        if cache == "e4m3":
            (c.k, c.ks), (c.v, c.vs) = R.quantise(k), R.quantise(v)
        else:
            c.k, c.v = k.bfloat16(), v.bfloat16()
        c.check(c.run())


def test_pages_outside_the_cache_and_lengths_past_the_table():
    c = Case([3, 3], [100, 90], seed=14)
    good = c.table.clone()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    c.check(c.run(err=err))
    assert int(err) == 0
    c.table[0, 2] = c.pages                                # one past the cache
    c.table[1, 1] = -1
    c.table[1, 5] = 1 << 30                                # the drafted tokens' page
    c.check(c.run(err=err))
    assert int(err) == 2
    c.run()                                                # without a word to tell it in
    c.table = good
    c.lengths = [100, 100000]                              # the table's pages past the length hold no page
    err.zero_()
    c.check(c.run(err=err))
    assert int(err) == 2
    c.lengths = [100, -3]
    err.zero_()
    c.check(c.run(err=err))
    assert int(err) == 0


def test_rows_of_no_request_are_left_as_they_were():
    c = Case([5, 2], [50, 300], heads=8, kv_heads=2, dim=64, tail=9, seed=15)
    a, k = c.args()
    out = torch.full_like(a[0], 7.0)
    lse = torch.full((16, 8), 7.0, device="cuda")
    attention.tree_attention(*a, **{**k, "out": out, "lse": lse})
    c.check((out, lse))
    assert bool((out[7:] == 7).all()) and bool((lse[7:] == 7).all())


def test_strided_queries_outputs_and_caches():
    """Queries out of a fused projection, an output transposed in memory, heads outside slots."""
    c = Case([7, 3], [200, 40], heads=8, kv_heads=4, dim=64, seed=16)
    a, k = c.args()
    wide = torch.zeros(10, 1024, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 256:768].view(10, 8, 64)
    q.copy_(a[0])
    out = torch.zeros(8, 10, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    both = torch.full((4, a[1].shape[0], 2, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    kc, vc = both[:, :, 0].transpose(0, 1), both[:, :, 1].transpose(0, 1)
    kc.copy_(a[1])
    vc.copy_(a[2])
    table = torch.zeros(2, 40, dtype=torch.int32, device="cuda")[:, :a[3].shape[1]]
    table.copy_(a[3])
    got = attention.tree_attention(q, kc, vc, table, a[4], **{**k, "out": out})
    assert got[0] is out
    c.check(got)


def test_offsets_past_32_bits():
    """Slots past 2^31 elements of the cache, and pages that end inside a tile."""
    heads, dim, page, slots = 8, 128, 16, (1 << 21) + 64
    kc, vc = (torch.empty(slots, heads, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = Case([4], [1000], heads=16, kv_heads=heads, dim=dim, page=page, seed=17)
    a, k = c.args()
    pages = slots // page
    table = torch.arange(pages - 63, pages, dtype=torch.int32, device="cuda").view(1, -1)
    pos = torch.arange(1000, device="cuda")
    new = table[0].long()[pos // page] * page + pos % page
    old = a[3][0].long()[pos // page] * page + pos % page
    kc[new], vc[new] = a[1][old], a[2][old]
    c.check(attention.tree_attention(a[0], kc, vc, table, a[4], **k))


def test_the_same_call_twice_gives_the_same_bits():
    c = Case([16, 4], [9000, 4000], heads=32, kv_heads=4, dim=128, cache="e4m3", tree=True, seed=18)
    a, k = c.args()
    first = attention.tree_attention(*a, **k)
    for _ in range(3):
        again = attention.tree_attention(*a, **k)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_lse_joins_two_parts_of_a_context():
    """The logsumexp is what joins attention over two halves of a context into the whole."""
    c = Case([1], [600], heads=8, kv_heads=2, dim=64, seed=19, kind="fp16", cache="fp16")
    a, k = c.args()
    whole, lse = attention.tree_attention(*a, **k)
    parts = []
    for lo, hi in ((0, 20), (20, 38)):
        n = torch.tensor([min(600, hi * 16) - lo * 16], dtype=torch.int32, device="cuda")
        parts.append(attention.tree_attention(a[0], a[1], a[2], a[3][:, lo:hi].contiguous(), n, **k))
    top = torch.logsumexp(torch.stack([p[1] for p in parts]), 0)
    joined = sum(p[0].float() * torch.exp(p[1] - top)[..., None] for p in parts)
    assert bool(((top - lse).abs() < 1e-4).all())
    # two parts and the whole, each rounded to fp16 and from fp16 weights: five half steps at most of |v| < 6
    assert bool(((joined - whole.float()).abs() < 5 * 2.0 ** -11 * 6).all())


def test_graphs_streams_and_workspaces():
    """Captured calls replay on new inputs; two graphs replay at once on two streams; a given workspace serves."""
    cases = [Case([16, 2], [5000, 700], heads=16, kv_heads=2, dim=128, seed=20 + i, cache="e4m3") for i in range(2)]
    held, graphs, outs = [], [], []
    for c in cases:
        a, k = c.args()
        held.append((a, k))
        attention.tree_attention(*a, **k)
    torch.cuda.synchronize()
    for a, k in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attention.tree_attention(*a, **k))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    want = [c.want() for c in cases]
    for c, o, w in zip(cases, outs, want):
        c.check(o, w)
    # new queries in the captured buffers
    cases[0].q = cases[1].q.clone()
    held[0][0][0].copy_(cases[0].q)
    graphs[0].replay()
    torch.cuda.synchronize()
    cases[0].check(outs[0])
    # a side stream and a workspace of one's own
    a, k = held[1]
    size = attention.workspace_bytes(16, 2, 128, 18)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")     # what it held before does not matter
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        got = attention.tree_attention(*a, **k, max_width=18, workspace=ws)
    streams[0].synchronize()
    cases[1].check(got, want[1])


def test_one_serving_round():
    """Rows written, attended over as a tree, the tree accepted, the kept slots' rows read back."""
    g = torch.Generator().manual_seed(30)
    B, T, heads, kv_heads, dim, slots = 3, 8, 8, 2, 64, 600
    prefix = torch.tensor([0, 100, 37], dtype=torch.int32)
    kc, vc, ks, vs = kvcache.allocate_kv(slots, kv_heads, dim, dtype=R.E4M3)
    table = torch.randperm(slots, generator=g)[:B * 150].view(B, 150).int()
    rows = [torch.randn(B * 150, kv_heads, dim, generator=g).bfloat16() for _ in range(2)]
    ctx = torch.cat([table[b, :int(prefix[b])] for b in range(B)])
    k, v = rows[0][:len(ctx)], rows[1][:len(ctx)]
    kvcache.write_kv(k.cuda(), v.cuda(), kc, vc, ctx.cuda(), k_scale=ks, v_scale=vs)
    draft = torch.cat([table[b, int(prefix[b]):int(prefix[b]) + T] for b in range(B)])
    dk, dv = rows[0][-B * T:], rows[1][-B * T:]
    kvcache.write_kv(dk.cuda(), dv.cuda(), kc, vc, draft.cuda(), k_scale=ks, v_scale=vs)
    parents = torch.tensor([_parents(g, T) for _ in range(B)])
    masks = attention.tree_mask(parents).cuda()
    q = torch.randn(B * T, heads, dim, generator=g).bfloat16()
    lens = (prefix + T).cuda()
    got = attention.tree_attention(q.cuda(), kc, vc, table.cuda(), lens, tree_mask=masks.view(-1), k_scale=ks, v_scale=vs,
                                   return_lse=True)
    want = R.attention(q, R.cache_values(kc, ks), R.cache_values(vc, vs), table, lens.tolist(), page_size=1,
                       starts=[0, T, 2 * T, 3 * T], masks=masks.view(-1).cpu(), scale=dim ** -0.5, group=heads // kv_heads, pages=slots)
    bound, _ = R.attention_bounds(*want, dim=dim, out_dtype=torch.bfloat16, weight_half_step=2.0 ** -11)
    assert bool(((got[0].double().cpu() - want[0]).abs() <= bound).all())
    top1 = torch.randint(0, 2, (B, T), generator=g).cuda()
    tokens = torch.randint(0, 2, (B, T), generator=g).cuda()
    r = accept.accept_tree(tokens, top1, masks, prefix_lens=prefix.cuda(), slots=draft.view(B, T).cuda())
    rk, rv = kvcache.read_kv(kc, vc, r.kept_slots.view(-1), k_scale=ks, v_scale=vs, dtype=torch.float32)
    codes, sc = R.quantise(dk)
    for b in range(B):
        path, out, bonus = R.accept(tokens[b].tolist(), top1[b].tolist(), parents[b].tolist())
        c = len(path)
        assert r.path[b, :c].tolist() == path and r.output[b, :c].tolist() == out and int(r.bonus[b]) == bonus
        at = torch.tensor([b * T + i for i in path])
        assert torch.equal(rk.view(B, T, kv_heads, dim)[b, :c].cpu(), codes.float()[at] * sc[at][..., None])
        assert not bool(rk.view(B, T, kv_heads, dim)[b, c:].any())


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("length", [129, 130, 133, 200, 100000, (1 << 31) - 1])
def test_a_length_past_the_table_leaves_the_drafted_tokens_where_they_are(length, tree):
    """The drafted tokens are the last of kv_lens also where the page table ends before them: the context keeps
    its positions, those past the table are unseen."""
    c = Case([5, 2], [128, 100], heads=8, kv_heads=2, dim=64, tree=tree, seed=21)
    if tree:
        c.masks[:5] = torch.tensor([0b1, 0b10, 0b100, 0b1001, 0b10000])
    c.lengths = [length, 100]
    c.table = c.table[:, :8].contiguous()                  # 128 positions
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = c.run(err=err)
    assert int(err) == 2
    # the same call with a table that goes on, with pages that are none (length: any at which all of it is context)
    c.lengths = [min(length, 300), 100]
    c.table = torch.cat([c.table, torch.full((2, 12), 1 << 30, dtype=torch.int32)], 1)
    c.check(got)


@pytest.mark.parametrize("length,page,kernels", [(64, 64, 1), (30, 16, 1), (65, 16, 2), (700, 16, 2)])
def test_the_kernels_of_a_call_are_counted(length, page, kernels):
    """One, and the one that joins items of more than one tile."""
    from dspine_b200 import _lib

    c = Case([1], [length], page=page, seed=22)
    a, k = c.args()
    table = a[3][:, :-(-length // page)].contiguous()
    before = _lib.load().dsv_launch_count()
    attention.tree_attention(a[0], a[1], a[2], table, a[4], **k)
    assert _lib.load().dsv_launch_count() - before == kernels
