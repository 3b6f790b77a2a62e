"""Oracle for the quantised paged KV cache and the attention over it: the definitions in 64 bits, on any device.

TEST INFRASTRUCTURE ONLY: the product never imports it.

A cache is uint8 [pages, kinds, heads, 64 * (D + 4)]: blocks of 64 tokens of D e4m3 bytes, then 64 f32 scales.
"""
from __future__ import annotations

import math

import torch

PAGE = 64
F8 = torch.float8_e4m3fn


def views(cache):
    """(e4m3 [pages, kinds, heads, 64, D], f32 scales [pages, kinds, heads, 64]) of a cache, no copies."""
    dim = cache.shape[-1] // PAGE - 4
    cache = cache.view(torch.uint8)
    return cache[..., : PAGE * dim].unflatten(-1, (PAGE, dim)).view(F8), cache[..., PAGE * dim:].view(torch.float32)


def rows(cache, slots, kind):
    """f64 [n, heads, D] of cache rows by slot; zeros for slots outside the cache."""
    values, scales = views(cache)
    slots = slots.long()
    there = (slots >= 0) & (slots < cache.shape[0] * PAGE)
    page, at = slots.clamp(0, cache.shape[0] * PAGE - 1) // PAGE, slots.clamp(0, cache.shape[0] * PAGE - 1) % PAGE
    x = values.view(torch.uint8)[page, kind, :, at].view(F8).double() * scales[page, kind, :, at].double()[..., None]
    return torch.where(there[:, None, None], x, 0.0)


def head_vectors(x, weight=None, cos_sin=None, positions=None, eps=1e-6, interleaved=False):
    """f64 [tokens, heads, D]: RMS norm of every head, then the first R dimensions turned by the position's row."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    if cos_sin is None:
        return x
    turn = cos_sin.double()[positions.long()][:, None]
    R = cos_sin.shape[1]
    cos, sin = turn[..., : R // 2], turn[..., R // 2:]
    i = torch.arange(R // 2, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    y = x.clone()
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., second] * cos + x[..., first] * sin
    return y


def random_cache(pages, kinds, heads, dim, seed=0, device="cpu"):
    """Quantised N(0, 0.5 .. 1.5) vectors."""
    g = torch.Generator(device=device).manual_seed(seed)
    cache = torch.empty(pages, kinds, heads, PAGE * (dim + 4), dtype=torch.uint8, device=device)
    values, scales = views(cache)
    values.view(torch.uint8).copy_((torch.randn(values.shape, generator=g, device=device) * 120).clamp(-448, 448).to(F8).view(torch.uint8))
    scales.copy_((0.5 + torch.rand(scales.shape, generator=g, device=device)) / 120)
    return cache


def attention(q, cache, block_table, seq_lens, q_starts, scale=None, window=0):
    """f64 (out, spread) [tokens, q_heads, D]; spread is the same average over |value|, the unit of rounding errors in the
    weights.  Rows of no sequence are NaN."""
    T, HQ, D = q.shape
    group = HQ // cache.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((T, HQ, D), float("nan"), dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
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
    return out, spread
