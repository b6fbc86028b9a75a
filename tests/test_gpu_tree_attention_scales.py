"""tree_attention over e4m3 caches whose V scales lie far apart."""

import math

import pytest
import torch

import kv_reference as R
from test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


def _slots(c, b, pos):
    pos = torch.as_tensor(pos)
    return c.table[b][pos // c.page].long() * c.page + pos % c.page


def _products_bound(c):
    """What rounding weight x V scale to fp16 may add to R.attention_bounds, [rows, heads, dim].

    The products of a row are held relative to the largest of those it sees, T, which lies in [2, 2^14]:
    one below fp16's normal numbers is off by up to half of its last step, 2^-25, so by 2^-26 T, times its code."""
    rows, heads, dim = c.q.shape
    codes, scales = c.v.float().double().nan_to_num(0.0), c.vs.double()
    k = R.cache_values(c.k, c.ks)
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    for b, n in enumerate(c.lengths):
        for r in range(c.starts[b], c.starts[b + 1]):
            own = torch.arange(n) - (n - c.widths[b])
            if c.masks is None:
                seen = own <= r - c.starts[b]
            else:
                bits = int(c.masks[r]) & (2 ** 64 - 1)
                seen = torch.tensor([j < 0 or bool(bits >> j & 1) for j in own.tolist()], dtype=torch.bool)
            at = _slots(c, b, torch.arange(n)[seen])
            x = torch.einsum("hd,lhd->hl", c.q[r].double(), k[at].repeat_interleave(c.group, 1)) * c.scale
            top = (torch.softmax(x, -1) * scales[at].abs().repeat_interleave(c.group, 1).t()).amax(-1)
            out[r] = 2.0 ** -26 * top[:, None] * codes[at].abs().sum(0).repeat_interleave(c.group, 0)
    return out


def _check(c, got):
    out, lse = (x.double().cpu() for x in got)
    want = c.want()
    bound, lse_bound = R.attention_bounds(*want, dim=c.q.shape[2], out_dtype=c.kind, weight_half_step=2.0 ** -11)
    bound = bound + _products_bound(c)
    off = (out - want[0]).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), "times the bound")
    off = (lse - want[1]).abs()
    assert bool((off <= lse_bound).all()), (float((off / lse_bound).max()), "times the bound of lse")


@pytest.mark.parametrize("kind,power", [("bf16", 20), ("bf16", 40), ("fp16", 20)])
def test_a_branch_with_a_large_value_does_not_touch_the_others(kind, power):
    """Two branches from a root; the nodes of the second have V scales far above all others."""
    c = Case([9, 1], [400, 200], heads=8, kv_heads=2, dim=128, kind=kind, cache="e4m3", tree=True, seed=1)
    first, second = [1, 2, 3, 4], [5, 6, 7, 8]
    c.masks[:9] = torch.tensor([1] + [1 | sum(1 << j for j in branch[:i + 1]) for branch in (first, second) for i in range(4)])
    if kind == "fp16":
        c.vs *= 2.0 ** -12                                 # both within fp16's range
    c.vs[_slots(c, 0, torch.arange(400 - 4, 400))] *= 2.0 ** power
    _check(c, c.run())


@pytest.mark.parametrize("power", [20, 40])
def test_later_tokens_of_a_chain_with_large_values(power):
    """Each drafted token's V is far above those before it: earlier rows do not see it."""
    c = Case([6, 3], [300, 90], heads=8, kv_heads=2, dim=64, cache="e4m3", seed=2)
    for j in range(6):
        c.vs[_slots(c, 0, [294 + j])] *= 2.0 ** (power * j / 5)
    _check(c, c.run())


@pytest.mark.parametrize("power,at", [(20, 0), (20, 250), (20, 699), (32, 3), (32, 650), (40, 130), (60, 350)])
def test_a_seen_value_of_next_to_no_weight_and_a_large_scale(power, at):
    """A key 2^-power below the others in weight whose V scale is 2^power above theirs: both count."""
    c = Case([2, 1], [702, 65], heads=4, kv_heads=1, dim=64, cache="e4m3", seed=3)
    c.q[..., 0] = 8.0
    slots = _slots(c, 0, torch.arange(702))
    c.k[slots, 0, 0] = torch.zeros(()).to(R.E4M3)
    c.k[slots[at], 0, 0] = torch.tensor(-448.0).to(R.E4M3)
    c.ks[slots[at], 0] = power * math.log(2.0) / 448.0      # scale 1/8 x 8 x this code: -power log 2 or so
    c.k[slots[at], 0, 1:] = torch.zeros(()).to(R.E4M3)
    c.vs[slots[at]] *= 2.0 ** power
    _check(c, c.run())


@pytest.mark.parametrize("dim,page,tree", [(128, 16, False), (64, 1, True), (80, 3, False)])
def test_scales_spread_over_40_powers_of_two(dim, page, tree):
    c = Case([5, 64, 1], [3000, 500, 130], heads=8, kv_heads=2, dim=dim, page=page, cache="e4m3", tree=tree, seed=4)
    g = torch.Generator().manual_seed(4)
    c.vs *= torch.exp2(40 * torch.rand(c.vs.shape, generator=g) - 20)
    _check(c, c.run())


@pytest.mark.parametrize("power", [-60, 90])
def test_scales_that_are_all_small_or_all_large(power):
    c = Case([3], [700], heads=4, kv_heads=2, dim=128, cache="e4m3", seed=5)
    c.vs *= 2.0 ** power
    _check(c, c.run())


@pytest.mark.parametrize("first", [True, False])
def test_small_scales_beside_very_large_ones(first):
    """Half of the context at 2^-70, half at 2^90: the weights of both halves count in the sum."""
    for length in (600, 4000):
        c = Case([1], [length], heads=4, kv_heads=2, dim=64, cache="e4m3", seed=6)
        half = torch.arange(length // 2)
        low, high = _slots(c, 0, half), _slots(c, 0, half + length // 2)
        if not first:
            low, high = high, low
        c.vs[low] *= 2.0 ** -70
        c.vs[high] *= 2.0 ** 90
        _check(c, c.run())


def test_scales_of_zero():
    """Scales of 0 (a row whose amax / 448 underflows) stand for zeros; the keys keep their weights."""
    c = Case([2, 1], [200, 70], heads=4, kv_heads=2, dim=64, cache="e4m3", seed=7)
    c.vs[_slots(c, 0, torch.arange(0, 200, 2))] = 0.0
    c.vs[_slots(c, 1, torch.arange(70))] = 0.0
    _check(c, c.run())


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dim,group", [(64, 4), (128, 20)])
def test_v_scales_that_are_not_finite_reach_the_rows_that_see_them(value, dim, group):
    """A drafted token with such a V scale: out of the rows that see it, no other row, and no logsumexp (which is K's)."""
    c = Case([6, 40, 2], [150, 60, 200], heads=2 * group, kv_heads=2, dim=dim, page=16, cache="e4m3", tree=True, seed=8, size=0.3)
    c.masks[:6] = torch.tensor([0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100001])
    c.vs[_slots(c, 0, [146]), 0] = value                   # node 2: rows 2 and 4
    c.vs[_slots(c, 1, [59]), 1] = value                    # node 39: itself, unless another row names it
    c.vs[_slots(c, 2, [3]), 0] = value                     # the context: every row
    c.masks[6:45] &= (1 << 39) - 1
    out, lse = (x.double().cpu() for x in c.run())
    want = c.want()
    _, lse_bound = R.attention_bounds(*want, dim=dim, out_dtype=c.kind, weight_half_step=2.0 ** -11)
    assert bool(torch.isfinite(lse).all()) and bool(((lse - want[1]).abs() <= lse_bound).all())
    touched = torch.zeros(48, 2, dtype=torch.bool)
    touched[[2, 4, 46, 47], 0] = True
    touched[45, 1] = True
    touched = touched.repeat_interleave(group, 1)
    assert torch.equal(~torch.isfinite(want[0]).all(-1), touched)
    same = out.nan_to_num(1.0, 2.0, 3.0) == want[0].nan_to_num(1.0, 2.0, 3.0)
    assert bool(same[touched].all())
    # the other rows' bounds, from a cache in which those tokens hold zeros (they do not see them)
    c.vs = torch.where(torch.isfinite(c.vs), c.vs, torch.zeros_like(c.vs))
    clean = c.want()
    bound, _ = R.attention_bounds(*clean, dim=dim, out_dtype=c.kind, weight_half_step=2.0 ** -11)
    assert bool(((out - clean[0]).abs() <= bound + _products_bound(c))[~touched].all())


@pytest.mark.parametrize("power,at", [(28, 299), (31, 310), (33, 257), (36, 500)])     # the first three in one tile
def test_fp16_values_of_next_to_no_weight(power, at):
    """An fp16 cache: one key carries the weight, another has 2^-power of it but 2^26 times its V."""
    c = Case([2, 1], [702, 65], heads=4, kv_heads=1, dim=64, kind="fp16", cache="fp16", seed=9)
    slots = _slots(c, 0, torch.arange(702))
    c.q[..., 0] = 8.0
    c.k[slots, 0] = 0.0
    c.k[slots, 0, 0] = -60 * math.log(2.0)                 # scale 1/8 x 8
    c.k[slots[300], 0, 0] = 0.0
    c.k[slots[at], 0, 0] = -(power + 0.53) * math.log(2.0)
    c.v[slots] = (c.v[slots].float() * 2.0 ** -10).half()
    c.v[slots[at]] = 60000.0
    out, lse = (x.double().cpu() for x in c.run())
    want = c.want()
    bound, lse_bound = R.attention_bounds(*want, dim=64, out_dtype=c.kind, weight_half_step=2.0 ** -11)
    # the row's largest weight lies in [2^9, 2^14]: one below fp16's normal numbers is off by up to 2^-25, so by 2^-34
    # of the largest (at most 1), times its value: 60000 of one key, 2^-8 at most of the 700 others
    bound[:2] += 2.0 ** -34 * (60000.0 + 700 * 2.0 ** -8)
    assert bool(((out - want[0]).abs() <= bound).all()), float(((out - want[0]).abs() / bound).max())
    assert bool(((lse - want[1]).abs() <= lse_bound).all())
