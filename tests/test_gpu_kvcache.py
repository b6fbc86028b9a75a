"""write_kv and read_kv on the GPU against their plain forms, bit for bit."""

import math

import pytest
import torch

from kv_reference import E4M3, quantise

from dspine_b200 import kvcache

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": E4M3}


def _rows(n, heads, dim, dtype, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g) * torch.exp(2 * torch.randn(n, heads, 1, generator=g))
    return x.to(dtype).to(device)


def _codes(x):
    return x.view(torch.uint8).cpu()


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,heads,dim,slots", [(1, 1, 16, 1), (3, 2, 64, 17), (100, 5, 80, 257), (1021, 8, 128, 4096),
                                               (33, 3, 256, 40), (7, 1, 112, 9)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_write_e4m3_is_the_quantisation_rule(kind, n, heads, dim, slots, index):
    k, v = _rows(n, heads, dim, TYPES[kind], 1), _rows(n, heads, dim, TYPES[kind], 2)
    k[n // 2, 0] = 0                                       # a row of zeros: scale 1
    kc, vc, ks, vs = kvcache.allocate_kv(slots, heads, dim, dtype=E4M3)
    kc.view(torch.uint8).fill_(0x55)
    ks.fill_(-3.0)
    at = torch.randperm(slots, generator=torch.Generator().manual_seed(3))[:n]
    kvcache.write_kv(k, v, kc, vc, at.to(index).cuda(), k_scale=ks, v_scale=vs)
    for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
        codes, scales = quantise(x)
        assert torch.equal(_codes(cache)[at], codes.view(torch.uint8))
        assert torch.equal(scale.cpu()[at], scales)
    rest = torch.ones(slots, dtype=torch.bool)
    rest[at] = False                                       # the other slots are left as they were
    assert bool((_codes(kc)[rest] == 0x55).all()) and bool((ks.cpu()[rest] == -3.0).all())


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,heads,dim", [(1, 1, 16), (65, 3, 96), (300, 8, 128), (9, 2, 256)])
def test_write_and_read_copy_rows_of_the_cache_type(kind, n, heads, dim):
    k, v = _rows(n, heads, dim, TYPES[kind], 4), _rows(n, heads, dim, TYPES[kind], 5)
    k[0, 0, 0], k[0, 0, 1] = math.inf, math.nan            # copied as they are
    kc, vc, _, _ = kvcache.allocate_kv(n + 5, heads, dim, dtype=TYPES[kind])
    at = torch.randperm(n + 5)[:n].int().cuda()
    kvcache.write_kv(k, v, kc, vc, at)
    assert torch.equal(kc[at.long()].view(torch.int16), k.view(torch.int16))
    assert torch.equal(vc[at.long()].view(torch.int16), v.view(torch.int16))
    for out in (torch.bfloat16, torch.float16, torch.float32):
        rk, rv = kvcache.read_kv(kc, vc, at, dtype=out)
        assert torch.equal(rv, v.float().to(out))
        assert torch.equal(torch.nan_to_num(rk, 7.0), torch.nan_to_num(k.float().to(out), 7.0))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
def test_read_every_code(out):
    """All 256 codes under scales of every size: code * scale in fp32, rounded once."""
    codes = torch.arange(256, dtype=torch.uint8).view(2, 1, 128).repeat(4, 3, 1)
    scales = torch.exp2(torch.arange(24).view(8, 3).float() * 2 - 20) * 1.37
    kc, ks = codes.cuda().view(E4M3), scales.cuda()
    slots = torch.tensor([5, 0, -1, 7, 5, 6, 1, 2, 3, 4], dtype=torch.int32, device="cuda")
    k, v = kvcache.read_kv(kc, kc.clone(), slots, k_scale=ks, v_scale=ks.clone(), dtype=out)
    want = (codes.view(E4M3).float() * scales[..., None])[slots.cpu().clamp(min=0).long()].to(out)
    want[2] = 0
    for got in (k, v):
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.cpu(), 0.0), torch.nan_to_num(want, 0.0))


def test_every_bf16_value_is_quantised_like_the_rule():
    """Every bf16 value against four row maxima: quotients on and beside the borders of all codes."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    every = every[torch.isfinite(every)]
    for top in (1.0, 448.0, 1.0078125, 3.3895e38):
        x = every[every.abs() <= torch.tensor(top).bfloat16()]
        x = torch.cat([x, x[:(-len(x)) % 120]]).view(-1, 1, 120)
        x = torch.cat([torch.full((len(x), 1, 8), top).bfloat16(), x], -1).contiguous()
        kc, vc, ks, vs = kvcache.allocate_kv(len(x), 1, 128, dtype=E4M3)
        kvcache.write_kv(x.cuda(), -x.cuda(), kc, vc, torch.arange(len(x), device="cuda"), k_scale=ks, v_scale=vs)
        for y, cache, scale in ((x, kc, ks), (-x, vc, vs)):
            codes, scales = quantise(y)
            assert torch.equal(scale.cpu(), scales)
            assert torch.equal(_codes(cache), codes.view(torch.uint8))


def test_random_fp32_rows_are_quantised_like_the_rule():
    x = _rows(4000, 2, 128, torch.float32, 8)
    kc, vc, ks, vs = kvcache.allocate_kv(4000, 2, 128, dtype=E4M3)
    kvcache.write_kv(x, x * 1e-30, kc, vc, torch.arange(4000, device="cuda"), k_scale=ks, v_scale=vs)
    for y, cache, scale in ((x, kc, ks), (x * 1e-30, vc, vs)):
        codes, scales = quantise(y)
        assert torch.equal(scale.cpu(), scales) and torch.equal(_codes(cache), codes.view(torch.uint8))


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_rows_of_every_size_are_quantised_like_the_rule(kind):
    """Row maxima from the smallest subnormals to the largest values: scales on every side of the
    range in which quotients come from a reciprocal, and quotients down to nothing."""
    g = torch.Generator().manual_seed(12)
    powers = torch.arange(-150, 127).repeat_interleave(8).double()
    n = len(powers)
    x = torch.randn(n, 1, 128, generator=g).double().clamp(-1.9, 1.9)
    x = x * torch.exp2(powers[:, None, None] - 12 * torch.rand(x.shape, generator=g).double())
    x = x.float().to(TYPES[kind])
    kc, vc, ks, vs = kvcache.allocate_kv(n, 1, 128, dtype=E4M3)
    kvcache.write_kv(x.cuda(), -x.cuda(), kc, vc, torch.arange(n, device="cuda"), k_scale=ks, v_scale=vs)
    for y, cache, scale in ((x, kc, ks), (-x, vc, vs)):
        codes, scales = quantise(y)
        assert torch.equal(scale.cpu(), scales)
        got, want = _codes(cache), codes.view(torch.uint8)
        # a scale that underflows to 0 makes 0 / 0, a NaN whose sign IEEE leaves open (0x7F and 0xFF are both NaN)
        both_nan = ((got & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F)
        assert bool(((got == want) | both_nan).all())


def test_rows_with_nan_infinity_and_tiny_values():
    x = torch.zeros(6, 1, 32)
    x[0, 0, 3], x[0, 0, 4] = math.nan, 2.0                 # scale 1, the NaN stays one
    x[1, 0, 5], x[1, 0, 6] = math.inf, 1.0                 # scale inf: inf / inf is NaN, 1 / inf is 0
    x[2, 0, 1], x[2, 0, 2] = 1e-40, -3e-41                 # subnormal
    x[3, 0, 0], x[3, 0, 1] = 3.4e38, 1e-30
    x[4] = torch.linspace(-1, 1, 32)
    kc, vc, ks, vs = kvcache.allocate_kv(6, 1, 32, dtype=E4M3)
    kvcache.write_kv(x.cuda(), x.cuda(), kc, vc, torch.arange(6, device="cuda"), k_scale=ks, v_scale=vs)
    codes, scales = quantise(x)
    assert torch.equal(ks.cpu(), scales) and torch.equal(vs.cpu(), scales)
    got, want = kc.cpu().float(), codes.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(got[0, 0, 3]))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_slots_outside_the_cache_are_skipped_and_told():
    k = _rows(6, 2, 64, torch.bfloat16, 9)
    kc, vc, ks, vs = kvcache.allocate_kv(4, 2, 64, dtype=E4M3)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.tensor([2, -1, 0, -7, 3, 1], device="cuda")
    kvcache.write_kv(k, k, kc, vc, slots, k_scale=ks, v_scale=vs, err=err)
    assert int(err) == 0                                   # a negative slot is padding
    before = _codes(kc).clone()
    slots = torch.tensor([4, 1 << 33, -1, -1, -1, -1], device="cuda")
    kvcache.write_kv(k, k, kc, vc, slots, k_scale=ks, v_scale=vs, err=err)
    assert int(err) == 1 and torch.equal(_codes(kc), before)
    err.zero_()
    rk, rv = kvcache.read_kv(kc, vc, slots, k_scale=ks, v_scale=vs, err=err)
    assert int(err) == 1 and not bool(rk.any()) and not bool(rv.any())
    kvcache.write_kv(k, k, kc, vc, slots, k_scale=ks, v_scale=vs)   # without a word to tell it in
    codes, _ = quantise(k)
    assert torch.equal(_codes(kc)[torch.tensor([2, 0, 3, 1])], codes.view(torch.uint8)[torch.tensor([0, 2, 4, 5])])


def test_strided_rows_and_caches():
    """Rows that are views of one projection, a cache with K and V interleaved, scales in a wider table."""
    n, heads, dim = 37, 4, 64
    qkv = _rows(n, 1, 3 * heads * dim, torch.bfloat16, 10)[:, 0]
    k = qkv[:, heads * dim:2 * heads * dim].view(n, heads, dim)
    v = qkv[:, 2 * heads * dim:].view(n, heads, dim)
    both = torch.zeros(50, 2, heads, dim, dtype=torch.uint8, device="cuda").view(E4M3)
    scales = torch.zeros(50, 2, heads, device="cuda")
    at = torch.randperm(50)[:n].cuda()
    kvcache.write_kv(k, v, both[:, 0], both[:, 1], at, k_scale=scales[:, 0], v_scale=scales[:, 1])
    for j, x in enumerate((k, v)):
        codes, sc = quantise(x)
        assert torch.equal(_codes(both[:, j])[at.cpu()], codes.view(torch.uint8))
        assert torch.equal(scales[:, j].cpu()[at.cpu()], sc)
    rk, rv = kvcache.read_kv(both[:, 0], both[:, 1], at, k_scale=scales[:, 0], v_scale=scales[:, 1], dtype=torch.float32)
    codes, sc = quantise(v)
    assert torch.equal(rv.cpu(), codes.float() * sc[..., None])
    # heads outside slots: [heads, slots, dim] storage seen as [slots, heads, dim]
    store = torch.zeros(2, heads, 50, dim, dtype=torch.bfloat16, device="cuda")
    kc, vc = store[0].transpose(0, 1), store[1].transpose(0, 1)
    kvcache.write_kv(k, v, kc, vc, at)
    assert torch.equal(store[1][:, at], v.transpose(0, 1))
    rk, rv = kvcache.read_kv(kc, vc, at)
    assert torch.equal(rk, k) and torch.equal(rv, v)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: its last slots, and the first."""
    heads, dim = 8, 128
    slots = (1 << 21) + 3
    kc, vc, ks, vs = (torch.empty(slots, heads, dim, dtype=torch.uint8, device="cuda").view(E4M3),
                      torch.empty(slots, heads, dim, dtype=torch.uint8, device="cuda").view(E4M3),
                      torch.empty(slots, heads, device="cuda"), torch.empty(slots, heads, device="cuda"))
    at = torch.tensor([slots - 1, 0, slots - 2, (1 << 21) - 1], device="cuda")
    k, v = _rows(4, heads, dim, torch.bfloat16, 11), _rows(4, heads, dim, torch.bfloat16, 12)
    kvcache.write_kv(k, v, kc, vc, at, k_scale=ks, v_scale=vs)
    rk, rv = kvcache.read_kv(kc, vc, at, k_scale=ks, v_scale=vs, dtype=torch.float32)
    for x, got, cache in ((k, rk, kc), (v, rv, vc)):
        codes, sc = quantise(x)
        assert torch.equal(cache[-1].view(torch.uint8).cpu(), codes.view(torch.uint8)[0])
        assert torch.equal(got.cpu(), codes.float() * sc[..., None])


def test_no_tokens_other_streams_and_graphs():
    k = _rows(8, 2, 64, torch.bfloat16, 13)
    kc, vc, ks, vs = kvcache.allocate_kv(16, 2, 64, dtype=E4M3)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    kvcache.write_kv(k[:0], k[:0], kc, vc, none, k_scale=ks, v_scale=vs)
    rk, rv = kvcache.read_kv(kc, vc, none, k_scale=ks, v_scale=vs)
    assert rk.shape == (0, 2, 64) and not bool(kc.view(torch.uint8).any())
    at = torch.arange(8, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        kvcache.write_kv(k, k, kc, vc, at, k_scale=ks, v_scale=vs)
        first = kvcache.read_kv(kc, vc, at, k_scale=ks, v_scale=vs, dtype=torch.float32)
    side.synchronize()
    codes, sc = quantise(k)
    assert torch.equal(first[0].cpu(), codes.float() * sc[..., None])
    g = torch.cuda.CUDAGraph()
    src, out = k.clone(), tuple(torch.zeros(8, 2, 64, dtype=torch.float32, device="cuda") for _ in range(2))
    with torch.cuda.graph(g):
        kvcache.write_kv(src, src, kc, vc, at, k_scale=ks, v_scale=vs)
        kvcache.read_kv(kc, vc, at, k_scale=ks, v_scale=vs, out=out)
    for seed in (14, 15):
        src.copy_(_rows(8, 2, 64, torch.bfloat16, seed))
        g.replay()
        torch.cuda.synchronize()
        codes, sc = quantise(src)
        assert torch.equal(out[1].cpu(), codes.float() * sc[..., None])
