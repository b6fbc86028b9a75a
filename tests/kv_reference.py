"""Plain 64-bit forms of the KV-cache and draft-tree operators, and the error bounds their
kernels are held to (arithmetic beside each)."""

import math

import torch

E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def quantise(x):
    """(codes, scales) of rows along the last dimension: scale amax / 448 (1 for a row of zeros or
    with a NaN), code = e4m3 of the fp32 quotient; on the CPU, where fp32 division is IEEE's."""
    x = x.float().cpu()
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, amax / torch.full_like(amax, 448.0), torch.ones_like(amax))
    y = x / scale[..., None]
    y = torch.where(torch.isnan(y), y, y.clamp(-448.0, 448.0))
    return y.to(E4M3), scale


def cache_values(cache, scale):
    """float64 values a cache stands for."""
    x = cache.cpu().to(torch.float32).double()
    return x if scale is None else x * scale.cpu().double()[..., None]


def attention(q, k, v, table, lens, *, page_size, starts, masks, scale, group, pages):
    """Per request: (out, lse, out bound terms) in float64 on the CPU, row by row over exactly the
    keys that it sees (so what a masked position holds cannot reach it).

    Returns out [rows, heads, dim], lse [rows, heads], absolute [rows, heads, dim] = sum p |v|,
    spread [rows, heads] = the largest sum_d |q_d k_d| * scale over the keys a row sees, and the
    longest length.  Rows outside every request are NaN."""
    q = q.cpu().double()
    n, heads, dim = q.shape
    out = torch.full((n, heads, dim), math.nan, dtype=torch.float64)
    absolute, lse = out.clone(), torch.full((n, heads), math.nan, dtype=torch.float64)
    spread = lse.clone()
    longest = 0
    for b in range(len(lens)):
        lo, hi = starts[b], starts[b + 1]
        length = min(max(int(lens[b]), 0), table.shape[1] * page_size)
        longest = max(longest, length)
        p0 = length - (hi - lo)
        page = table[b].long().cpu()
        for r in range(lo, hi):
            i = r - lo
            pos = torch.arange(length)
            own = pos - p0
            if masks is None:
                seen = own <= i
            else:
                bits = int(masks[r]) & (2 ** 64 - 1)
                seen = torch.tensor([j < 0 or (j < 64 and bool(bits >> j & 1)) for j in own.tolist()], dtype=torch.bool)
            pos = pos[seen]
            at = page[pos // page_size]
            ok = (at >= 0) & (at < pages)
            slot = at[ok] * page_size + pos[ok] % page_size
            if len(slot) == 0:
                out[r], lse[r], absolute[r], spread[r] = 0.0, -math.inf, 0.0, 0.0
                continue
            kk = k[slot].repeat_interleave(group, 1)        # [L, heads, dim]
            vv = v[slot].repeat_interleave(group, 1)
            x = torch.einsum("hd,lhd->hl", q[r], kk) * scale
            p = torch.softmax(x, -1)
            out[r] = torch.einsum("hl,lhd->hd", p, vv)
            absolute[r] = torch.einsum("hl,lhd->hd", p, vv.abs())
            lse[r] = torch.logsumexp(x, -1)
            spread[r] = (torch.einsum("hd,lhd->hl", q[r].abs(), kk.abs()) * scale).amax(-1)
    return out, lse, absolute, spread, longest


def attention_bounds(out, lse, absolute, spread, longest, *, dim, out_dtype, weight_half_step):
    """Elementwise bounds on the kernel's out and lse.

    A score is a sum of dim products in fp32, then scaled: off by at most (dim + 8) 2^-23 times the
    sum of their sizes (dim + 8 roundings or truncations of at most one step); the exponential is
    approximated to 2^-21 (ex2.approx: 2^-22, its argument rounded twice).  So a weight is off by
    a relative d = spread (dim + 8) 2^-23 + 2^-21, its normaliser by the same, the sums over keys
    by (longest / 16 + 160) 2^-23 (accumulated in steps of 16 keys, then joined).  Weights are
    rounded to the operand type once (weight_half_step), the result to out_dtype once."""
    d = spread * (dim + 8) * 2.0 ** -23 + 2.0 ** -21
    total = 2 * d + (longest / 16 + 160) * 2.0 ** -23 * 2
    # the smallest subnormal of the output type bounds roundings near zero
    tiny = 2.0 ** -24 if out_dtype == torch.float16 else 1e-37
    bound = HALF_STEP[out_dtype] * out.abs() + (weight_half_step + total)[..., None] * absolute * 1.01 + tiny
    return bound, total + 2.0 ** -22 * (1 + lse.abs().nan_to_num(0.0, 0.0, 0.0))


def accept(tokens, top1, parents):
    """One tree, walked from its root: (path, output tokens, bonus)."""
    n = len(tokens)
    if n == 0:
        return [], [], -1
    depth, good = [0] * n, [False] * n
    for i in range(n):
        if i == 0:
            good[0] = True
            continue
        p = parents[i]
        depth[i] = depth[p] + 1 if p >= 0 else 0
        good[i] = p >= 0 and good[p] and tokens[i] == top1[p]
    best = max((i for i in range(n) if good[i]), key=lambda i: (depth[i], -i))
    path = []
    i = best
    while i >= 0:
        path.append(i)
        i = parents[i] if i > 0 else -1
    path.reverse()
    return path, [tokens[i] for i in path[1:]] + [top1[best]], top1[best]
