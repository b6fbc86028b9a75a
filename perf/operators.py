"""The KV-cache and draft-tree operators as cases that can be measured.

Four operators of one serving round, in the order they run: the drafted tokens' keys and values
are written into a slot-addressed cache (quantised to e4m3 or kept), the drafted tokens attend
over the cached context and over their own ancestors in the draft tree, the accepted path of the
tree is found from the target's top-1 tokens, and cached rows are read back.

`run(state)` computes one of them: in plain 32-bit torch operations, or, where `own` is true,
through the package's entry points.  `exact(case, seed)` is the same from the definitions in 64
bits, request by request.
"""

import math

import numpy as np
import torch

own = False

E4M3 = torch.float8_e4m3fn
KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": E4M3}


# ---- the cases -----------------------------------------------------------------------------

def listed():
    return [
        # one user, one new token on a short context: the smallest call, all latency
        {"name": "attend 1x1 short", "op": "attend", "requests": 1, "width": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "longest": 333, "page": 16, "kind": "bf16", "cache": "bf16", "tree": False},
        # ordinary decoding without drafts: a full batch of single tokens on ragged contexts
        {"name": "attend 64x1 bf16", "op": "attend", "requests": 64, "width": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "longest": 8192, "page": 16, "kind": "bf16", "cache": "bf16", "tree": False},
        # verification of 16-token draft chains, ragged widths, e4m3 cache, one slot per page
        {"name": "attend 64x16 chain e4m3", "op": "attend", "requests": 64, "width": 16, "heads": 32, "kv_heads": 8, "dim": 128,
         "longest": 4096, "page": 1, "kind": "bf16", "cache": "e4m3", "tree": False},
        # trees of up to 64 nodes under many query heads: the most arithmetic per cached byte
        {"name": "attend 16x64 tree bf16", "op": "attend", "requests": 16, "width": 64, "heads": 64, "kv_heads": 8, "dim": 128,
         "longest": 16384, "page": 64, "kind": "bf16", "cache": "bf16", "tree": True},
        # one very long context: few rows, the work has to be split along the cache
        {"name": "attend 1x16 long e4m3", "op": "attend", "requests": 1, "width": 16, "heads": 32, "kv_heads": 4, "dim": 128,
         "longest": 131071, "page": 16, "kind": "bf16", "cache": "e4m3", "tree": False},
        # a small model in fp16: odd sizes, 7 query heads per key head, narrow heads, small trees
        {"name": "attend 7x13 tree fp16", "op": "attend", "requests": 7, "width": 13, "heads": 14, "kv_heads": 2, "dim": 64,
         "longest": 1021, "page": 8, "kind": "fp16", "cache": "fp16", "tree": True},
        # the rows of one verification round of 64 requests x 16 drafted tokens
        {"name": "write 1024 e4m3", "op": "write", "tokens": 1024, "kv_heads": 8, "dim": 128, "slots": 65536,
         "kind": "bf16", "cache": "e4m3"},
        # the rows of a long prompt
        {"name": "write 32749 e4m3", "op": "write", "tokens": 32749, "kv_heads": 8, "dim": 128, "slots": 65536,
         "kind": "bf16", "cache": "e4m3"},
        # a block of one request's cache read back
        {"name": "read 1000 e4m3", "op": "read", "tokens": 1000, "kv_heads": 8, "dim": 128, "slots": 65536,
         "kind": "bf16", "cache": "e4m3"},
        # a whole context read back, to be sent elsewhere or recomputed on
        {"name": "read 131072 e4m3", "op": "read", "tokens": 131072, "kv_heads": 8, "dim": 128, "slots": 262144,
         "kind": "bf16", "cache": "e4m3"},
        # the accepted path of a few small trees
        {"name": "accept 4x16", "op": "accept", "requests": 4, "width": 16},
        # the largest round: 256 requests, trees of up to 64 nodes
        {"name": "accept 256x64", "op": "accept", "requests": 256, "width": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "accept"])
    if op == "attend":
        kind = rng.choice(["bf16", "bf16", "fp16"])
        width = rng.choice([1, _log(rng, 2, 16), _log(rng, 2, 64)])
        kv_heads = rng.choice([1, 2, 4, 8])
        c = {"op": op, "requests": _log(rng, 1, 64), "width": width, "heads": kv_heads * rng.choice([1, 2, 4, 5, 7, 8]),
             "kv_heads": kv_heads, "dim": rng.choice([64, 80, 96, 128, 128]), "longest": 1, "page": rng.choice([1, 8, 16, 64]),
             "kind": kind, "cache": rng.choice([kind, "e4m3"]), "tree": rng.random() < 0.5}
        # as long as it may be without costing more than the largest listed case
        top = min(131072, int(min(64 * 8 * 8192 / (c["requests"] * kv_heads), 16 * 64 * 64 * 16384 / (c["requests"] * c["heads"] * width))))
        c["longest"] = max(width, _log(rng, max(2, min(200, top // 2)), top))
        return c
    if op == "accept":
        return {"op": op, "requests": _log(rng, 1, 256), "width": _log(rng, 2, 64)}
    c = {"op": op, "tokens": _log(rng, 1, 32768 if op == "write" else 131072), "kv_heads": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 80, 96, 128, 128]), "slots": 0, "kind": rng.choice(["bf16", "fp16"]), "cache": "e4m3"}
    if rng.random() < 0.25:
        c["cache"] = c["kind"]
    c["slots"] = c["tokens"] + _log(rng, 1, 65536)
    return c


# ---- sizes that follow from a case alone ---------------------------------------------------

def _widths(case):
    """Drafted tokens of each request: all of them one where the width is 1, else ragged with the widest first."""
    w = case["width"]
    return [max(1, w - int((b * 0.6180339887) % 1.0 * 0.75 * w)) for b in range(case["requests"])]


def _lengths(case):
    """Cached tokens of each request, its drafted ones among them: ragged, the longest first."""
    return [max(w, int(round(case["longest"] * (1.0 - 0.9 * ((b * 0.7548776662) % 1.0)))))
            for b, w in enumerate(_widths(case))]


def work(case):
    if case["op"] == "accept":
        n = sum(_widths(case))
        return {"bytes": n * (8 + 8 + 8 + 4) + case["requests"] * (case["width"] * (8 + 4 + 4) + 28), "flops": 0}
    size = {"bf16": 2, "fp16": 2, "e4m3": 1}
    row = case["kv_heads"] * case["dim"]
    held = row * size[case["cache"]] + (4 * case["kv_heads"] if case["cache"] == "e4m3" else 0)
    if case["op"] in ("write", "read"):
        return {"bytes": case["tokens"] * (2 * (row * 2 + held) + 4), "flops": 0}
    n, q = sum(_widths(case)), case["heads"] * case["dim"]
    keys = sum(_lengths(case))
    seen = sum(w * n for w, n in zip(_widths(case), _lengths(case)))
    return {"bytes": keys * (2 * held + 4 / case["page"]) + n * (2 * 2 * q + 4 * case["heads"]), "flops": 4 * seen * q}


# ---- inputs --------------------------------------------------------------------------------

def _trees(rng, widths):
    """Ancestor bits of random draft trees, node by node: bit j of node i is set where j is i or an ancestor of i.
    Drafters branch near the root and then follow their best candidates, so most nodes hang from a recent one."""
    masks, parents = [], []
    for w in widths:
        own_masks = [1]
        parents.append(-1)
        for i in range(1, w):
            p = i - 1 - min(i - 1, int(rng.exponential(2.0)))
            parents.append(p)
            own_masks.append(own_masks[p] | (1 << i))
        masks += own_masks
    return np.array(masks, dtype=np.uint64).view(np.int64), np.array(parents)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _quantised(x):
    """e4m3 codes and scales of the rows of x, as the write operator defines them."""
    amax = x.float().abs().amax(-1)
    scale = torch.where(amax > 0, amax / torch.full_like(amax, 448.0), torch.ones_like(amax))
    return (x.float() / scale[..., None]).clamp(-448.0, 448.0).to(E4M3), scale


def _rows(g, n, heads, dim, kind):
    """Keys or values as a model makes them: channels of different spread and mean, around one in size."""
    spread = torch.exp(0.4 * torch.randn(heads, dim, device="cuda", generator=g))
    mean = 0.5 * torch.randn(heads, dim, device="cuda", generator=g)
    return (torch.randn(n, heads, dim, device="cuda", generator=g) * spread + mean).to(KINDS[kind])


def _cached(g, slots, heads, dim, kind, cache):
    x = _rows(g, slots, heads, dim, kind)
    return _quantised(x) if cache == "e4m3" else (x, None)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    if case["op"] == "accept":
        return _prepare_accept(case, rng)
    heads, dim, kind = case["kv_heads"], case["dim"], case["kind"]
    if case["op"] in ("write", "read"):
        s = {"op": case["op"], "kind": KINDS[kind],
             "slots": torch.randperm(case["slots"], device="cuda", generator=g)[:case["tokens"]].int()}
        s["k_cache"], s["k_scale"] = _cached(g, case["slots"], heads, dim, kind, case["cache"])
        s["v_cache"], s["v_scale"] = _cached(g, case["slots"], heads, dim, kind, case["cache"])
        if case["op"] == "write":
            s["k"] = _rows(g, case["tokens"], heads, dim, kind)
            s["v"] = _rows(g, case["tokens"], heads, dim, kind)
        return s
    widths, lengths, page = _widths(case), _lengths(case), case["page"]
    pages = [-(-n // page) for n in lengths]
    total = sum(pages) + 3
    order = torch.randperm(total, device="cuda", generator=g).int()
    table = torch.zeros(len(pages), max(pages), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"op": "attend", "table": table, "page": page, "width": case["width"],
         "lengths": _cuda(np.array(lengths, dtype=np.int32)),
         "starts": _cuda(np.concatenate([[0], np.cumsum(widths)]).astype(np.int32)),
         "masks": _cuda(_trees(rng, widths)[0]) if case["tree"] else None,
         "scale": 1.0 / math.sqrt(dim),
         "q": torch.randn(sum(widths), case["heads"], dim, device="cuda", generator=g).to(KINDS[kind])}
    s["k_cache"], s["k_scale"] = _cached(g, total * page, heads, dim, kind, case["cache"])
    s["v_cache"], s["v_scale"] = _cached(g, total * page, heads, dim, kind, case["cache"])
    return s


def _prepare_accept(case, rng):
    """Trees whose nodes agree with the target's top-1 token of their parent four times in five."""
    widths = _widths(case)
    masks, parents = _trees(rng, widths)
    starts = np.concatenate([[0], np.cumsum(widths)])
    first = np.repeat(starts[:-1], widths)
    top1 = rng.randint(0, 151936, size=len(masks)).astype(np.int64)
    tokens = rng.randint(0, 151936, size=len(masks)).astype(np.int64)
    agree = (parents >= 0) & (rng.rand(len(masks)) < 0.8)
    tokens[agree] = top1[(first + parents)[agree]]
    return {"op": "accept", "tokens": _cuda(tokens), "top1": _cuda(top1), "masks": _cuda(masks), "width": case["width"],
            "starts": _cuda(starts.astype(np.int32)), "prefix": _cuda(rng.randint(1, 8192, size=len(widths)).astype(np.int32)),
            "slots": _cuda(rng.permutation(131072)[:len(masks)].astype(np.int32))}


# ---- one pass ------------------------------------------------------------------------------

def run(s):
    return {"attend": _attend, "write": _write, "read": _read, "accept": _accept}[s["op"]](s)


def _attend(s):
    if own:
        from dspine_b200 import attention

        out, lse = attention.tree_attention(
            s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], page_size=s["page"], q_indptr=s["starts"],
            max_width=s["width"], tree_mask=s["masks"], scale=s["scale"], k_scale=s["k_scale"], v_scale=s["v_scale"],
            return_lse=True)
        return {"out": out, "lse": lse}
    q, starts, lengths, page, t = s["q"], s["starts"].long(), s["lengths"].long(), s["page"], s["width"]
    n, heads, dim = q.shape
    kv_heads = s["k_cache"].shape[1]
    group, b, dev = heads // kv_heads, lengths.numel(), q.device
    pos = torch.arange(s["table"].shape[1] * page, device=dev)
    slot = s["table"].long()[:, pos // page] * page + pos % page                       # [B, L]
    slot = torch.where(pos < lengths[:, None], slot, torch.zeros_like(slot))
    k = s["k_cache"].view(torch.uint8)[slot].view(s["k_cache"].dtype).float() if s["k_scale"] is not None else s["k_cache"][slot].float()
    v = s["v_cache"].view(torch.uint8)[slot].view(s["v_cache"].dtype).float() if s["v_scale"] is not None else s["v_cache"][slot].float()
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][slot][..., None], v * s["v_scale"][slot][..., None]
    i = torch.arange(t, device=dev)
    widths = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + i).clamp(max=n - 1)                                     # [B, T]
    real = i < widths[:, None]
    drafted = pos - (lengths - widths)[:, None]                                        # [B, L]: place in the draft
    if s["masks"] is None:
        seen = drafted[:, None] <= i[:, None]
    else:
        seen = (drafted < 0)[:, None] | ((s["masks"][row][:, :, None] >> drafted.clamp(0, 63)[:, None]) & 1).bool()
    seen = (seen & (pos < lengths[:, None])[:, None])[:, None, :, None]                # [B, 1, T, 1, L]
    qr = q[row].float().view(b, t, kv_heads, group, dim).permute(0, 2, 1, 3, 4)        # [B, Hkv, T, G, D]
    x = torch.matmul(qr.reshape(b, kv_heads, t * group, dim), k.permute(0, 2, 3, 1)) * s["scale"]
    x = x.view(b, kv_heads, t, group, -1).masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, kv_heads, t * group, -1), v.transpose(1, 2)).view(b, kv_heads, t, group, dim)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    lse = (torch.log(total) + m)[..., 0]
    out = o.permute(0, 2, 1, 3, 4).reshape(b, t, heads, dim)[real].to(q.dtype)
    return {"out": out, "lse": lse.permute(0, 2, 1, 3).reshape(b, t, heads)[real]}


def _write(s):
    if own:
        from dspine_b200 import kvcache

        kvcache.write_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    else:
        at = s["slots"].long()
        if s["k_scale"] is None:
            s["k_cache"][at], s["v_cache"][at] = s["k"], s["v"]
        else:
            for x, cache, scale in ((s["k"], "k_cache", "k_scale"), (s["v"], "v_cache", "v_scale")):
                codes, scales = _quantised(x)
                s[cache].view(torch.uint8)[at] = codes.view(torch.uint8)
                s[scale][at] = scales
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _read(s):
    if own:
        from dspine_b200 import kvcache

        k, v = kvcache.read_kv(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"], dtype=s["kind"])
        return {"k": k, "v": v}
    at = s["slots"].long()
    if s["k_scale"] is None:
        return {"k": s["k_cache"][at], "v": s["v_cache"][at]}
    k = s["k_cache"].view(torch.uint8)[at].view(E4M3).float() * s["k_scale"][at][..., None]
    v = s["v_cache"].view(torch.uint8)[at].view(E4M3).float() * s["v_scale"][at][..., None]
    return {"k": k.to(s["kind"]), "v": v.to(s["kind"])}


def _accept(s):
    if own:
        from dspine_b200 import accept

        r = accept.accept_tree(s["tokens"], s["top1"], s["masks"], q_indptr=s["starts"], prefix_lens=s["prefix"],
                               slots=s["slots"], width=s["width"])
        return {"accept": r.accept, "commit": r.commit, "bonus": r.bonus, "output": r.output, "path": r.path,
                "kept_slots": r.kept_slots, "new_seq": r.new_seq}
    t, starts = s["width"], s["starts"].long()
    dev = starts.device
    i = torch.arange(t, device=dev)
    real = i < (starts[1:] - starts[:-1])[:, None]
    row = (starts[:-1, None] + i).clamp(max=s["tokens"].numel() - 1)
    above = (s["masks"][row][:, :, None] >> i) & 1                                     # [B, T, T]: ancestors and itself
    above = above.bool() & (i[:, None] >= i)
    strict = above & (i[:, None] > i)
    parent = torch.where(strict, i, torch.full_like(i, -1)).amax(-1)                   # [B, T]
    top1, tokens = s["top1"][row], s["tokens"][row]
    agree = (i == 0) | ((parent >= 0) & (tokens == torch.gather(top1, 1, parent.clamp(min=0))))
    good = real & (~above | agree[:, None, :]).all(-1) & above[:, :, 0]
    depth = above.sum(-1)
    best = torch.where(good, depth * t + (t - 1 - i), torch.full_like(depth, -1)).argmax(-1, keepdim=True)   # deepest, then first
    on = torch.gather(above, 1, best[..., None].expand(-1, -1, t))[:, 0]               # [B, T]: nodes of the path
    commit = on.sum(-1)
    path = torch.sort(torch.where(on, i, torch.full_like(i, t)), -1).values
    held = i < commit[:, None]
    bonus = torch.gather(top1, 1, best)[:, 0]
    after = torch.cat([path[:, 1:], path[:, :1]], 1).clamp(max=t - 1)
    output = torch.where(i < (commit - 1)[:, None], torch.gather(tokens, 1, after), torch.zeros_like(tokens))
    output = torch.where(i == (commit - 1)[:, None], bonus[:, None], output)
    kept = torch.gather(s["slots"][row], 1, path.clamp(max=t - 1))
    none = torch.full_like(path, -1)
    return {"accept": (commit - 1).int(), "commit": commit.int(), "bonus": bonus, "output": output,
            "path": torch.where(held, path, none).int(), "kept_slots": torch.where(held, kept, none.int()),
            "new_seq": s["prefix"] + commit.int()}


# ---- from the definitions, in 64 bits ------------------------------------------------------

def _held(cache, scale, at):
    x = cache.view(torch.uint8)[at].view(E4M3).double() if scale is not None else cache[at].double()
    return x if scale is None else x * scale[at].double().unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "accept":
        return None  # whole numbers
    if s["op"] == "read":
        at = s["slots"].long()
        return {"k": _held(s["k_cache"], s["k_scale"], at), "v": _held(s["v_cache"], s["v_scale"], at)}
    if s["op"] == "write":
        got = {}
        at = s["slots"].long()
        for n in ("k", "v"):
            cache, scale, x = s[n + "_cache"].double(), s[n + "_scale"], s[n].double()
            if scale is None:
                cache[at] = x
                got[n + "_scale"] = None
            else:
                top = x.abs().amax(-1, keepdim=True)
                step = torch.where(top > 0, top / 448.0, torch.ones_like(top))
                y = x / step                                   # |y| <= 448; e4m3: 3 bits after the leading one, 2^-9 at least
                e = torch.frexp(y)[1].clamp(min=-5) - 4
                cache[at] = torch.round(y * torch.exp2(-e.double())) * torch.exp2(e.double())
                scale = scale.double()
                scale[at] = step[..., 0]
                got[n + "_scale"] = scale
            got[n + "_cache"] = cache
        return got
    if work(case)["flops"] > 2e13:
        return None
    outs, sums = [], []
    starts, lengths, page = s["starts"].tolist(), s["lengths"].tolist(), s["page"]
    q = s["q"].double()
    group = q.shape[1] // s["k_cache"].shape[1]
    for b, n in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        w = hi - lo
        pos = torch.arange(n, device=q.device)
        at = s["table"][b].long()[pos // page] * page + pos % page
        k = _held(s["k_cache"], s["k_scale"], at).repeat_interleave(group, 1)
        v = _held(s["v_cache"], s["v_scale"], at).repeat_interleave(group, 1)
        x = torch.einsum("thd,lhd->htl", q[lo:hi], k) * s["scale"]
        own_rows = torch.ones(w, w, dtype=torch.bool, device=q.device).tril()
        if s["masks"] is not None:
            own_rows = ((s["masks"][lo:hi, None] >> torch.arange(w, device=q.device)) & 1).bool()
        x[:, :, n - w:] = torch.where(own_rows, x[:, :, n - w:], torch.full_like(x[:, :, n - w:], -math.inf))
        p = torch.softmax(x, -1)
        outs.append(torch.einsum("htl,lhd->thd", p, v))
        sums.append(torch.logsumexp(x, -1).t())
    return {"out": torch.cat(outs), "lse": torch.cat(sums)}
