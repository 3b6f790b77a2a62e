"""Oracle for the paged KV cache in 4 bits and the attention over it: the definitions in 64 bits, on any device.

TEST INFRASTRUCTURE ONLY: the product never imports it.

A cache is uint8 [pages, 2, heads, 64 * (D / 2 + D / 16 + 4)]: D / 64 planes of [64 tokens, 32 bytes] of e2m1 codes, then [64, D / 16]
e4m3 group scales, then 64 f32 scales.  Norm and rotation are the 8-bit cache's (:func:`kv_oracle.head_vectors`).
"""
from __future__ import annotations

import math

import torch

PAGE, GROUP = 64, 16
F8 = torch.float8_e4m3fn
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def dim_of(cache):
    return {2560: 64, 4864: 128}[cache.shape[-1]]


def views(cache):
    """(code bytes [pages, 2, heads, D / 64, 64, 32], group scales' bytes [pages, 2, heads, 64, D / 16], f32 scales [pages, 2, heads, 64])
    of a cache, no copies."""
    dim = dim_of(cache)
    cache = cache.view(torch.uint8)
    a, b = 32 * dim, 36 * dim
    return cache[..., :a].unflatten(-1, (dim // 64, PAGE, 32)), cache[..., a:b].unflatten(-1, (PAGE, dim // GROUP)), cache[..., b:].view(torch.float32)


def parts(cache, slots, kind):
    """(codes [n, heads, D], group scales f64 [n, heads, D / 16], scales f64 [n, heads]) of rows that are there."""
    codes, groups, scales = views(cache)
    page, at = slots.long() // PAGE, slots.long() % PAGE
    b = codes[page, kind, :, :, at].long()
    return (torch.stack([b % 16, b // 16], dim=-1).flatten(-3), groups[page, kind, :, at].view(F8).double(), scales[page, kind, :, at].double())


def rows(cache, slots, kind):
    """f64 [n, heads, D] of cache rows by slot; zeros for slots outside the cache."""
    slots = slots.long()
    there = (slots >= 0) & (slots < cache.shape[0] * PAGE)
    codes, groups, scales = parts(cache, slots.clamp(0, cache.shape[0] * PAGE - 1), kind)
    table = torch.tensor(VALUES, dtype=torch.float64, device=cache.device)
    x = table[codes] * groups.repeat_interleave(GROUP, dim=-1) * scales[..., None]
    return torch.where(there[:, None, None], x, 0.0)


def nearest_codes(x):
    """e2m1 codes of x (f64): nearest, the even code between two, at most 6."""
    magnitudes = torch.tensor(VALUES[:8], dtype=torch.float64, device=x.device)
    a = x.abs().clamp(max=6.0)
    distance = (a[..., None] - magnitudes).abs()
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)      # even codes first: the first of equal distances
    code = order[distance[..., order].argmin(-1)]
    return code + 8 * (x < 0)


def quantised(z):
    """(codes, group scales, scales) of head vectors z [..., D] with every operation in f32, as the definition says."""
    z = z.float()
    scale = (z.abs().amax(-1).clamp(min=float(torch.tensor(1e-12))).double() / 2688.0).float()     # (on a GPU torch divides f32 by a number with its reciprocal)
    group = (z.abs().unflatten(-1, (-1, GROUP)).amax(-1).double() / (6.0 * scale).double()[..., None]).float().to(F8)
    unit = (group.float() * scale[..., None]).repeat_interleave(GROUP, dim=-1)
    quotient = torch.where(unit > 0, (z.double() / unit.double()).float(), 0.0)
    return nearest_codes(quotient.double()), group.double(), scale.double()


def random_cache(pages, heads, dim, seed=0, device="cpu"):
    """Quantised N(0, 0.5 .. 1.5) vectors."""
    g = torch.Generator(device=device).manual_seed(seed)
    cache = torch.empty(pages, 2, heads, PAGE * (dim // 2 + dim // GROUP + 4), dtype=torch.uint8, device=device)
    codes, groups, scales = views(cache)
    x = torch.randn(*codes.shape, 2, generator=g, device=device) * 2.7
    magnitude = sum((x.abs() > border).to(torch.uint8) for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
    magnitude += 8 * (x < 0).to(torch.uint8)
    codes.copy_(magnitude[..., 0] + 16 * magnitude[..., 1])
    groups.copy_((448.0 * (0.35 + 0.65 * torch.rand(groups.shape, generator=g, device=device))).to(F8).view(torch.uint8))
    scales.copy_((0.5 + torch.rand(scales.shape, generator=g, device=device)) / 800)
    return cache


def attention(q, cache, block_table, seq_lens, q_starts, scale=None, window=0):
    """f64 (out, spread, floor) [tokens, q_heads, D]; spread is the same average over |value|, the unit of rounding errors in the
    weights.  floor is 2^-28 of the row's largest product of weight and value scale, times the sum of |code * group scale|: what the sums
    are off by where every weight is off by so much (the interface lets a weight 2^-28 below the largest be left out).  Rows of no
    sequence are NaN."""
    T, HQ, D = q.shape
    group = HQ // cache.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((T, HQ, D), float("nan"), dtype=torch.float64, device=q.device)
    spread, floor = torch.zeros_like(out), torch.zeros_like(out)
    for b, length in enumerate(seq_lens.tolist()):
        lo, hi = int(q_starts[b]), int(q_starts[b + 1])
        if lo == hi:
            continue
        length = max(0, min(length, block_table.shape[1] * PAGE))
        j = torch.arange(length, device=q.device)
        entry = block_table[b].long()[j // PAGE]
        there = (entry >= 0) & (entry < cache.shape[0])
        j, slots = j[there], (entry * PAGE + j % PAGE)[there]
        keys, values = rows(cache, slots, 0), rows(cache, slots, 1)
        table = torch.tensor(VALUES[:8], dtype=torch.float64, device=q.device)
        codes, groups, scales = parts(cache, slots, 1)
        units = (table[codes % 8] * groups.repeat_interleave(GROUP, dim=-1)).nan_to_num(0.0)
        p = (torch.arange(lo, hi, device=q.device) - hi + length)[:, None]
        seen = j <= p
        if window:
            seen &= j > p - window
        for h in range(HQ):
            x = (q[lo:hi, h].double() @ keys[:, h // group].T * scale).masked_fill(~seen, -math.inf)
            top = x.amax(-1, keepdim=True) if len(j) else torch.zeros(hi - lo, 1, dtype=torch.float64, device=q.device)
            w = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
            total = w.sum(-1, keepdim=True)
            w = torch.where(seen, w / torch.where(total == 0, 1.0, total), 0.0)
            v = values[:, h // group]
            # a row's own positions only: what it does not see may be anything
            clean = torch.where(v.isfinite(), v, 0.0)
            out[lo:hi, h] = w @ clean
            for bad in (~v.isfinite()).any(-1).nonzero()[:, 0].tolist():
                out[lo:hi, h][seen[:, bad]] = float("nan")
            spread[lo:hi, h] = w @ clean.abs()
            if len(j):
                largest = (w * scales[:, h // group].nan_to_num(0.0, 0.0)).amax(-1, keepdim=True)
                floor[lo:hi, h] = 2.0 ** -28 * largest * (seen.double() @ units[:, h // group])
    return out, spread, floor
