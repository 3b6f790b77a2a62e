"""The quantised paged KV cache and the attention over it, as cases that can be timed: writing new tokens' keys and values
(head norms, rotation, quantisation and the scatter in one call), reading rows back by slot, and attention of new tokens
(one per sequence, chunks, whole prompts) over the cache.

The cache is bytes [pages, 2 (keys, values) or 1 (keys only), kv heads, 64 * (D + 4)]: 64 tokens of D e4m3 bytes, then their 64
f32 scales.  ``run`` computes the operators in plain torch operations in 32 bits, or, where ``own`` is true, calls the
framework.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
PAGE = 64
F8 = torch.float8_e4m3fn
EPS = 1e-6
_package = None


def _pkg():
    global _package
    if _package is None:
        _package = importlib.import_module("mlsys-contest-syfi-agent-assisted_b200")
    return _package


# ------------------------------------------------------------------------------------------------- the cases
def _write(name, tokens, q_heads, kv_heads, dim=128, rotary=128, norm=True, interleaved=False, padded=0):
    """q_heads = 0: a cache of keys only (what an index of a sequence's tokens keeps)."""
    case = {"op": "write", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "norm": norm, "interleaved": interleaved, "padded": padded}
    return dict(case, name=name) if name else case


def _read(name, rows, kv_heads, dim=128, missing=0):
    case = {"op": "read", "rows": rows, "kv_heads": kv_heads, "dim": dim, "missing": missing}
    return dict(case, name=name) if name else case


def _attention(name, batch, q_short, q_long, kv_short, kv_long, q_heads, kv_heads, dim=128, window=0):
    """Lengths of the sequences' new tokens and of the whole sequences, see _lengths."""
    case = {"op": "attention", "batch": batch, "q_short": q_short, "q_long": q_long, "kv_short": kv_short, "kv_long": kv_long,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "window": window}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a decode step's new tokens, one for each of 24 sequences
        _write("write_t24", 24, 32, 8),
        # index keys of a prefill chunk: one key head, half of its dimensions rotated, a chunk padded to its graph's size
        _write("write_index_t1000", 1000, 0, 1, rotary=64, padded=13),
        # the large prefill of the benchmark
        _write("write_t8192", 8192, 64, 8),
        # the 2048 tokens that an indexer keeps of a sequence, not all there
        _read("read_selected", 2048, 8, missing=300),
        # a long prefix brought back for a kernel that wants bf16
        _read("read_t40000", 40000, 8),
        # one short sequence being decoded: latency
        _attention("attn_b1_short", 1, 1, 1, 700, 700, 32, 8),
        # a decode batch with the lengths of the indexer's ordinary one
        _attention("attn_b24_ragged", 24, 1, 1, 300, 30000, 32, 8),
        # a decode batch of long sequences: two million tokens
        _attention("attn_b32_64k", 32, 1, 1, 65536, 65536, 32, 4),
        # decoding and chunks of prompts in one batch, as a scheduler packs them
        _attention("attn_mixed_b8", 8, 1, 250, 500, 12000, 32, 8),
        # a chunk of a prompt behind a long context, narrow heads
        _attention("attn_chunk_t512", 1, 512, 512, 40000, 40000, 32, 4, dim=64),
        # two chunks with one key head for all 64 query heads, each query sees the last 1024 positions
        _attention("attn_window_b2", 2, 700, 1100, 5000, 6001, 64, 1, window=1024),
        # a whole prompt of the benchmark's prefill size
        _attention("attn_prefill_t8192", 1, 8192, 8192, 8192, 8192, 32, 8),
    ]


MOST_SCORES = 32 * 8192 * 8192          # of a padded batch: the largest listed prompt
MOST_BYTES = 2 * 32 * 65536 * 4 * 132   # of cache: the largest listed decode batch


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    return rng.choice([(32, 8), (32, 8), (32, 4), (64, 8), (16, 16), (64, 1), (24, 8), (12, 4), (40, 8), (8, 8)])


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk", "prompt"])
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice([128, 128, 64])
    if kind == "write":
        keys_only = rng.random() < 0.25
        tokens = _log_uniform(rng, 1, 8192)
        rotary = rng.choice([dim, dim, dim // 2])
        return _write(None, tokens, 0 if keys_only else q_heads, 1 if keys_only else kv_heads, dim, rotary, rng.random() < 0.7,
                      rng.random() < 0.3, rng.randrange(1 + tokens // 8))
    if kind == "read":
        rows = _log_uniform(rng, 1, 40000)
        return _read(None, rows, min(kv_heads, 8), dim, rng.choice([0, rows // 7]))
    if kind == "decode":
        batch = _log_uniform(rng, 1, 64)
        kv_long = _log_uniform(rng, 17, min(65536, MOST_BYTES // (batch * kv_heads * 2 * (dim + 4))))
        kv_short = _log_uniform(rng, max(2, kv_long // 100), kv_long)
        q = rng.choice([1, 1, 1, 2, 5])
        return _attention(None, batch, 1, q, kv_short, kv_long, q_heads, kv_heads, dim, rng.choice([0, 0, 0, 700]))
    if kind == "chunk":
        batch = _log_uniform(rng, 1, 12)
        q_long = _log_uniform(rng, 10, 2000 if batch < 4 else 500)
        kv_long = _log_uniform(rng, q_long, max(q_long, min(50000, MOST_SCORES // (batch * q_heads * q_long))))
        kv_short = _log_uniform(rng, max(1, kv_long // 20), kv_long)
        return _attention(None, batch, _log_uniform(rng, 1, q_long), q_long, kv_short, kv_long, q_heads, kv_heads, dim,
                          rng.choice([0, 0, 512, 4096]))
    batch = rng.choice([1, 1, 2, 3])
    kv_long = _log_uniform(rng, 100, int(math.sqrt(MOST_SCORES / (batch * q_heads))))
    kv_short = _log_uniform(rng, max(1, kv_long // 10), kv_long)
    return _attention(None, batch, kv_short, kv_long, kv_short, kv_long, q_heads, kv_heads, dim, rng.choice([0, 0, 0, 1000]))


def _spread(n, a, b):
    """n lengths from a to b, evenly over the logarithm."""
    return [b] if n == 1 else [int(round(a * (b / a) ** (i / (n - 1)))) for i in range(n)]


def _lengths(case):
    """(new tokens, whole length) of each sequence: a prompt's are equal, else the longest chunks lie in the middle of the context lengths."""
    n = case["batch"]
    kv = _spread(n, case["kv_short"], case["kv_long"])
    q = _spread(n, case["q_short"], case["q_long"])
    if (case["q_short"], case["q_long"]) != (case["kv_short"], case["kv_long"]):
        q = q[n // 2:] + q[:n // 2]
    return [min(a, b) for a, b in zip(q, kv)], kv


# ------------------------------------------------------------------------------------------------- the inputs
def _random_cache(g, pages, kinds, heads, dim):
    """Keys and values as a quantisation by token and head leaves them: e4m3 values whose largest are near 448, f32 scales."""
    cache = torch.empty(pages, kinds, heads, PAGE * (dim + 4), dtype=torch.uint8, device=DEV)
    values, scales = _views(cache, dim)
    step = max(1, (1 << 28) // (kinds * heads * PAGE * dim))
    for at in range(0, pages, step):
        part = values[at: at + step]
        part.copy_((torch.randn(part.shape, generator=g, device=DEV) * 120.0).clamp_(-448.0, 448.0).to(F8).view(torch.uint8))
    scales.copy_((0.5 + torch.rand(scales.shape, generator=g, device=DEV)) / 120.0)
    return cache


def _views(cache, dim):
    """(bytes [pages, kinds, heads, 64, D], scales [pages, kinds, heads, 64]) of a cache, without a copy."""
    return cache[..., : PAGE * dim].unflatten(-1, (PAGE, dim)), cache[..., PAGE * dim:].view(torch.float32)


def _prepare_write(case, g):
    T, HQ, HK, D, R = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "rotary"))
    # what a fused projection leaves: queries, keys and values side by side in a token's row
    kinds = 2 if HQ else 1
    fused = torch.randn(T, (HQ + kinds * HK) * D, generator=g, device=DEV)
    fused *= 0.3 + torch.rand(T, 1, generator=g, device=DEV)
    fused = fused.to(torch.bfloat16)
    q = fused[:, : HQ * D].unflatten(-1, (HQ, D)) if HQ else None
    k = fused[:, HQ * D: (HQ + HK) * D].unflatten(-1, (HK, D))
    v = fused[:, (HQ + HK) * D:].unflatten(-1, (HK, D)) if HQ else None
    weights = [(1.0 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) if case["norm"] else None for _ in range(2)]
    longest = T + 5000
    angle = torch.arange(longest, device=DEV).double()[:, None] * 10000.0 ** (-torch.arange(0, R, 2, device=DEV).double() / R)
    cos_sin = torch.cat([angle.cos(), angle.sin()], dim=-1).float()
    first = int(torch.randint(0, 5000, (1,), generator=g, device=DEV))
    positions = torch.arange(first, first + T, dtype=torch.int32, device=DEV)
    pages = (T + PAGE - 1) // PAGE + 2
    place = torch.randperm(pages, generator=g, device=DEV)
    at = torch.arange(T, device=DEV) + 17           # the first page is partly full
    slots = (place[at // PAGE] * PAGE + at % PAGE).to(torch.int32)
    if case["padded"]:
        slots[T - case["padded"]:] = -1
    cache = _random_cache(g, pages, kinds, HK, D)
    q_out = torch.empty(T, HQ, D, dtype=torch.bfloat16, device=DEV) if HQ else None
    return {"q": q, "k": k, "v": v, "q_weight": weights[0] if HQ else None, "k_weight": weights[1], "cos_sin": cos_sin,
            "positions": positions, "slots": slots, "cache": cache, "q_out": q_out, "interleaved": case["interleaved"]}


def _prepare_read(case, g):
    n, H, D = case["rows"], case["kv_heads"], case["dim"]
    pages = (n + n // 4) // PAGE + 2
    cache = _random_cache(g, pages, 2, H, D)
    slots = torch.randperm(pages * PAGE, generator=g, device=DEV)[:n].to(torch.int32)
    if case["missing"]:
        slots[n - case["missing"]:] = -1
    out = [torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    return {"cache": cache, "slots": slots, "k_out": out[0], "v_out": out[1], "dim": D}


def _prepare_attention(case, g):
    HQ, HK, D = case["q_heads"], case["kv_heads"], case["dim"]
    q_lens, kv_lens = _lengths(case)
    need = [(n + PAGE - 1) // PAGE for n in kv_lens]
    pages, width = sum(need) + 3, max(need) + 2
    cache = _random_cache(g, pages, 2, HK, D)
    place = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)      # every sequence's pages lie scattered over the cache
    table = torch.zeros(case["batch"], width, dtype=torch.int32)
    host, at = place.cpu(), 0
    for b, n in enumerate(need):
        table[b, :n] = host[at: at + n]
        at += n
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1], HQ, D, generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    return {"q": q, "cache": cache, "table": table.to(DEV), "seq_lens": torch.tensor(kv_lens, dtype=torch.int32, device=DEV),
            "q_starts": torch.tensor(starts, dtype=torch.int32, device=DEV), "out": torch.empty_like(q), "window": case["window"],
            "longest_q": max(q_lens)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    state = {"write": _prepare_write, "read": _prepare_read, "attention": _prepare_attention}[case["op"]](case, g)
    return dict(state, op=case["op"])


# ------------------------------------------------------------------------------------------------- one pass
def _rotated(x, cos_sin, interleaved):
    """x [T, H, D], cos_sin [T, R]: the first R dimensions turned, pairs (i, i + R/2) or (2 i, 2 i + 1)."""
    R = cos_sin.shape[-1]
    cos, sin = cos_sin[:, None, : R // 2], cos_sin[:, None, R // 2:]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., : R // 2], x[..., R // 2: R])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, dim=-1).flatten(-2) if interleaved else torch.cat(turned, dim=-1)
    return torch.cat([turned, x[..., R:]], dim=-1)


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.to(x.dtype)


def _put(values, scales, kind, slots, x):
    there = (slots >= 0).nonzero()[:, 0]
    page, at, x = slots[there] // PAGE, slots[there] % PAGE, x[there]
    scale = x.abs().amax(-1).clamp_min(1e-12) / 448.0
    values[page, kind, :, at] = (x / scale[..., None]).to(F8).view(torch.uint8)
    scales[page, kind, :, at] = scale


def _write_outputs(cache, dim, q_out):
    values, scales = _views(cache, dim)
    return {"values": values.view(F8), "scales": scales, "q": q_out}


def _run_write(s):
    dim = s["k"].shape[-1]
    if own:
        _pkg().run_kv_write(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"], s["slots"],
                            s["cache"], s["q_out"], eps=EPS, interleaved=s["interleaved"])
        return _write_outputs(s["cache"], dim, s["q_out"])
    turn = s["cos_sin"][s["positions"]]
    values, scales = _views(s["cache"], dim)
    _put(values, scales, 0, s["slots"], _rotated(_normed(s["k"].float(), s["k_weight"]), turn, s["interleaved"]))
    if s["q"] is not None:
        _put(values, scales, 1, s["slots"], s["v"].float())
        s["q_out"].copy_(_rotated(_normed(s["q"].float(), s["q_weight"]), turn, s["interleaved"]))
    return _write_outputs(s["cache"], dim, s["q_out"])


def _run_read(s):
    if own:
        _pkg().run_kv_read(s["cache"], s["slots"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    values, scales = _views(s["cache"], s["dim"])
    page, at = s["slots"].clamp_min(0) // PAGE, s["slots"].clamp_min(0) % PAGE
    rows = values[page, :, :, at].view(F8).float() * scales[page, :, :, at][..., None]      # [n, 2, heads, D]
    rows = torch.where((s["slots"] >= 0)[:, None, None, None], rows, 0.0).to(torch.bfloat16)
    return rows[:, 0], rows[:, 1]


def _run_attention(s):
    q, window = s["q"], s["window"]
    if own:
        return _pkg().run_paged_attention(q, s["cache"], s["table"], s["seq_lens"], s["q_starts"], s["out"], window=window)
    (T, HQ, D), HK, B = q.shape, s["cache"].shape[2], len(s["seq_lens"])
    Q, G = s["longest_q"], HQ // HK
    n_q = s["q_starts"][1:] - s["q_starts"][:-1]
    values, scales = _views(s["cache"][s["table"]], D)                                      # [B, pages, 2, heads, 64, D]
    kv = (values.view(F8).float() * scales[..., None]).permute(2, 0, 3, 1, 4, 5).flatten(3, 4)   # [2, B, heads, tokens, D]
    i = torch.arange(Q, device=q.device)
    rows = (s["q_starts"][:-1, None] + i).clamp_max(T - 1)
    grouped = q[rows].float().unflatten(2, (HK, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)    # [B, heads, Q G, D]
    x = torch.matmul(grouped, kv[0].transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).unflatten(2, (Q, G))
    position = (s["seq_lens"] - n_q)[:, None, None] + i[None, :, None]                      # [B, Q, 1]
    j = torch.arange(kv.shape[3], device=q.device)
    hidden = j > position
    if window:
        hidden |= j <= position - window
    x.masked_fill_(hidden[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    x = torch.matmul(x.flatten(2, 3), kv[1]).unflatten(2, (Q, G)) / torch.where(total > 0, total, 1.0)
    t = torch.arange(T, device=q.device)
    b = torch.searchsorted(s["q_starts"][1:], t, right=True)
    return x.permute(0, 2, 1, 3, 4)[b, t - s["q_starts"][b]].flatten(1, 2).to(torch.bfloat16)    # [T, HQ, D]


def run(state):
    return {"write": _run_write, "read": _run_read, "attention": _run_attention}[state["op"]](state)


# ------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    D = case["dim"]
    if case["op"] == "write":
        T, HQ, HK = case["tokens"], case["q_heads"], case["kv_heads"]
        kinds, kept = (2 if HQ else 1), T - case["padded"]
        vectors = T * HQ + kept * kinds * HK
        size = vectors * D * 2 + T * (case["rotary"] * 4 + 8) + T * HQ * D * 2 + kept * kinds * HK * (D + 4)
        return {"bytes": size, "flops": vectors * D * 8}
    if case["op"] == "read":
        rows, there = case["rows"] * case["kv_heads"] * 2, (case["rows"] - case["missing"]) * case["kv_heads"] * 2
        return {"bytes": there * (D + 4) + rows * D * 2 + case["rows"] * 4, "flops": there * D}
    window, read, seen = case["window"], 0, 0
    q_lens, kv_lens = _lengths(case)
    for n, length in zip(q_lens, kv_lens):
        first = length - n
        read += min(length, n + window - 1) if window else length
        if window:
            short = max(0, min(window, length) - first)       # queries with fewer positions than the window
            seen += sum(range(first + 1, first + short + 1)) + (n - short) * window
        else:
            seen += n * first + n * (n + 1) // 2
    return {"bytes": sum(q_lens) * case["q_heads"] * D * 4 + read * case["kv_heads"] * 2 * (D + 4),
            "flops": 4 * D * case["q_heads"] * seen}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _exact_vectors(x, weight, cos_sin, interleaved):
    """The definition's head vectors of x [T, H, D] in 64 bits: norm, then each pair as a complex number times cos + i sin."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    if cos_sin is None:
        return x
    R = cos_sin.shape[-1]
    first = torch.arange(0, R, 2, device=x.device) if interleaved else torch.arange(R // 2, device=x.device)
    second = first + (1 if interleaved else R // 2)
    turn = torch.complex(cos_sin[:, : R // 2].double(), cos_sin[:, R // 2:].double())[:, None]
    z = torch.complex(x[..., first], x[..., second]) * turn
    x = x.clone()
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_write(s):
    dim = s["k"].shape[-1]
    turn = s["cos_sin"][s["positions"].long()]
    values = _views(s["cache"], dim)[0].view(F8).double()
    scales = _views(s["cache"], dim)[1].double()
    written = [_exact_vectors(s["k"], s["k_weight"], turn, s["interleaved"])]
    if s["v"] is not None:
        written.append(_exact_vectors(s["v"], None, None, False))
    slots = s["slots"].long()
    for kind, x in enumerate(written):
        for t in range(0, len(slots), 1024):
            part = slots[t: t + 1024]
            keep = part >= 0
            page, at, y = part[keep] // PAGE, part[keep] % PAGE, x[t: t + 1024][keep]
            scale = y.abs().amax(-1).clamp(min=1e-12) / 448.0
            values[page, kind, :, at] = y / scale[..., None]
            scales[page, kind, :, at] = scale
    q = None if s["q"] is None else _exact_vectors(s["q"], s["q_weight"], turn, s["interleaved"])
    return {"values": values, "scales": scales, "q": q}


def _exact_tokens(s, slots, dim):
    """(keys, values) [n, heads, D] in 64 bits of cache rows."""
    values, scales = _views(s["cache"], dim)
    page, at = slots // PAGE, slots % PAGE
    return [values[page, kind, :, at].view(F8).double() * scales[page, kind, :, at].double()[..., None] for kind in range(2)]


def _exact_read(s):
    slots = s["slots"].long()
    return tuple(torch.where((slots >= 0)[:, None, None], x, 0.0) for x in _exact_tokens(s, slots.clamp(min=0), s["dim"]))


def _exact_attention(s):
    T, HQ, D = s["q"].shape
    starts, lengths = s["q_starts"].tolist(), s["seq_lens"].tolist()
    out = torch.zeros(T, HQ, D, dtype=torch.float64, device=DEV)
    for b, length in enumerate(lengths):
        lo, hi = starts[b], starts[b + 1]
        j = torch.arange(length, device=DEV)
        keys, values = _exact_tokens(s, s["table"][b].long()[j // PAGE] * PAGE + j % PAGE, D)
        group = HQ // keys.shape[1]
        for h in range(HQ):
            k, v = keys[:, h // group], values[:, h // group]
            for at in range(lo, hi, 2048):
                to = min(hi, at + 2048)
                p = (torch.arange(at, to, device=DEV) - hi + length)[:, None]
                seen = (j <= p) & (j > p - s["window"]) if s["window"] else j <= p
                x = (s["q"][at:to, h].double() @ k.T) / math.sqrt(D)
                out[at:to, h] = torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1) @ v
    return out


def exact(case, seed):
    state = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attention": _exact_attention}[case["op"]](state)
