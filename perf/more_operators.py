"""A paged KV cache held in 4 bits and the attention over it, as cases that can be timed: writing new tokens' keys and values (head
norms, rotation, quantisation and the scatter in one call), reading rows back by slot, and attention of new tokens (one per sequence,
chunks, whole prompts) over the cache.

The cache is bytes [pages, 2 (keys, values), kv heads, 64 * (D / 2 + D / 16 + 4)]: D / 64 planes of 64 dimensions, each of 64 tokens'
e2m1 codes, two to a byte (the even dimension in the low half); then the 64 tokens' D / 16 e4m3 group scales; then their f32 scales.
A value is code * group scale * scale.
``run`` computes the operators in plain torch operations in 32 bits, or, where ``own`` is true, calls the framework.
"""
import importlib
import math

import torch

own = False

DEV = "cuda:0"
PAGE, GROUP = 64, 16
F8 = torch.float8_e4m3fn
EPS = 1e-6
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)       # of the codes 0 .. 7; 8 .. 15 are the same below zero
_package = None
_tables = {}


def _pkg():
    global _package
    if _package is None:
        _package = importlib.import_module("mlsys-contest-syfi-agent-assisted_b200")
    return _package


def _table(kind):
    """What the codes stand for: "values" f32 [16]; "pairs" int16 [256], both codes of a byte as two e4m3 bytes."""
    if kind not in _tables:
        values = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=DEV)
        byte = torch.arange(256, device=DEV)
        pairs = torch.stack([values[byte % 16], values[byte // 16]], dim=-1).to(F8)
        _tables.update(values=values, pairs=pairs.view(torch.int16)[:, 0].contiguous())
    return _tables[kind]


# ------------------------------------------------------------------------------------------------- the cases
def _write(name, tokens, q_heads, kv_heads, dim=128, rotary=128, norm=True, interleaved=False, padded=0):
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
        _write("write4_t24", 24, 32, 8),
        # a prefill chunk padded to its graph's size, narrow heads of which half is rotated in neighbouring pairs
        _write("write4_t1000", 1000, 24, 8, dim=64, rotary=32, norm=False, interleaved=True, padded=13),
        # the large prefill of the benchmark
        _write("write4_t8192", 8192, 64, 8),
        # the 2048 tokens that an indexer keeps of a sequence, not all there
        _read("read4_selected", 2048, 8, missing=300),
        # a long prefix brought back for a kernel that wants bf16
        _read("read4_t40000", 40000, 8),
        # one short sequence being decoded: latency
        _attention("attn4_b1_short", 1, 1, 1, 700, 700, 32, 8),
        # a decode batch with the lengths of the indexer's ordinary one
        _attention("attn4_b24_ragged", 24, 1, 1, 300, 30000, 32, 8),
        # a decode batch of long sequences: two million tokens
        _attention("attn4_b32_64k", 32, 1, 1, 65536, 65536, 32, 4),
        # decoding and chunks of prompts in one batch, as a scheduler packs them
        _attention("attn4_mixed_b8", 8, 1, 250, 500, 12000, 32, 8),
        # a chunk of a prompt behind a long context, narrow heads
        _attention("attn4_chunk_t512", 1, 512, 512, 40000, 40000, 32, 4, dim=64),
        # two chunks with one key head for all 64 query heads, each query sees the last 1024 positions
        _attention("attn4_window_b2", 2, 700, 1100, 5000, 6001, 64, 1, window=1024),
        # a whole prompt of the benchmark's prefill size
        _attention("attn4_prefill_t8192", 1, 8192, 8192, 8192, 8192, 32, 8),
    ]


MOST_SCORES = 32 * 8192 * 8192          # of a padded batch: the largest listed prompt
MOST_VECTORS = 2 * 32 * 65536 * 4       # of cache: the largest listed decode batch


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    return rng.choice([(32, 8), (32, 8), (32, 4), (64, 8), (16, 16), (64, 1), (24, 8), (12, 4), (40, 8), (8, 8)])


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk", "prompt"])
    q_heads, kv_heads = _heads(rng)
    dim = rng.choice([128, 128, 64])
    if kind == "write":
        tokens = _log_uniform(rng, 1, 8192)
        rotary = rng.choice([dim, dim, dim // 2])
        return _write(None, tokens, q_heads, kv_heads, dim, rotary, rng.random() < 0.7, rng.random() < 0.3, rng.randrange(1 + tokens // 8))
    if kind == "read":
        rows = _log_uniform(rng, 1, 40000)
        return _read(None, rows, min(kv_heads, 8), dim, rng.choice([0, rows // 7]))
    if kind == "decode":
        batch = _log_uniform(rng, 1, 64)
        kv_long = _log_uniform(rng, 17, min(65536, MOST_VECTORS // (batch * kv_heads * 2)))
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
def _views(cache, dim):
    """(bytes [pages, 2, heads, D / 64, 64, 32], e4m3 [pages, 2, heads, 64, D / 16], f32 [pages, 2, heads, 64]) of a cache, without a copy."""
    a, b = PAGE * dim // 2, PAGE * dim // 2 + PAGE * dim // GROUP
    return (cache[..., :a].unflatten(-1, (dim // 64, PAGE, 32)), cache[..., a:b].unflatten(-1, (PAGE, dim // GROUP)).view(F8),
            cache[..., b:].view(torch.float32))


def _codes(x):
    """e2m1 codes of x: the nearest value, the one with an even code between two, at most 6."""
    a = x.abs()
    code = (a > 0.25).to(torch.uint8)
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border) if up else (a > border)
    return code + 8 * (x < 0).to(torch.uint8)


def _random_cache(g, pages, heads, dim):
    """Keys and values as a quantisation leaves them: codes up to 6, group scales that spread below 448, f32 scales by token and head."""
    cache = torch.empty(pages, 2, heads, PAGE * (dim // 2 + dim // GROUP + 4), dtype=torch.uint8, device=DEV)
    codes, groups, scales = _views(cache, dim)
    step = max(1, (1 << 27) // (2 * heads * PAGE * dim))
    for at in range(0, pages, step):
        part = codes[at: at + step]
        c = _codes(torch.randn(*part.shape, 2, generator=g, device=DEV) * 2.7)
        part.copy_(c[..., 0] + 16 * c[..., 1])
    groups.copy_((448.0 * (0.35 + 0.65 * torch.rand(groups.shape, generator=g, device=DEV))).to(F8))
    scales.copy_((0.5 + torch.rand(scales.shape, generator=g, device=DEV)) / 800.0)
    return cache


def _prepare_write(case, g):
    T, HQ, HK, D, R = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "rotary"))
    # what a fused projection leaves: queries, keys and values side by side in a token's row
    fused = torch.randn(T, (HQ + 2 * HK) * D, generator=g, device=DEV)
    fused *= 0.3 + torch.rand(T, 1, generator=g, device=DEV)
    fused = fused.to(torch.bfloat16)
    q, k, v = (x.unflatten(-1, (-1, D)) for x in fused.split([HQ * D, HK * D, HK * D], dim=-1))
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
    _table("pairs")
    return {"q": q, "k": k, "v": v, "q_weight": weights[0], "k_weight": weights[1], "cos_sin": cos_sin, "positions": positions,
            "slots": slots, "cache": _random_cache(g, pages, HK, D), "q_out": torch.empty(T, HQ, D, dtype=torch.bfloat16, device=DEV),
            "interleaved": case["interleaved"]}


def _prepare_read(case, g):
    n, H, D = case["rows"], case["kv_heads"], case["dim"]
    pages = (n + n // 4) // PAGE + 2
    slots = torch.randperm(pages * PAGE, generator=g, device=DEV)[:n].to(torch.int32)
    if case["missing"]:
        slots[n - case["missing"]:] = -1
    out = [torch.empty(n, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    return {"cache": _random_cache(g, pages, H, D), "slots": slots, "k_out": out[0], "v_out": out[1], "dim": D}


def _prepare_attention(case, g):
    HQ, HK, D = case["q_heads"], case["kv_heads"], case["dim"]
    q_lens, kv_lens = _lengths(case)
    need = [(n + PAGE - 1) // PAGE for n in kv_lens]
    pages, width = sum(need) + 3, max(need) + 2
    cache = _random_cache(g, pages, HK, D)
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


def _put(cache, kind, slots, x):
    codes, groups, scales = _views(cache, x.shape[-1])
    there = (slots >= 0).nonzero()[:, 0]
    page, at, x = slots[there] // PAGE, slots[there] % PAGE, x[there].unflatten(-1, (-1, GROUP))
    scale = x.abs().amax((-1, -2)).clamp_min(1e-12) / 2688.0
    group = (x.abs().amax(-1) / (6.0 * scale)[..., None]).to(F8)
    unit = (group.float() * scale[..., None])[..., None]
    c = _codes(torch.where(unit > 0, x / unit, 0.0)).flatten(-2)
    codes[page, kind, :, :, at] = (c[..., 0::2] + 16 * c[..., 1::2]).unflatten(-1, (-1, 32))
    groups.view(torch.uint8)[page, kind, :, at] = group.view(torch.uint8)
    scales[page, kind, :, at] = scale


def _write_outputs(cache, dim, q_out):
    codes, groups, scales = _views(cache, dim)
    values = torch.index_select(_table("pairs"), 0, codes.int().flatten()).view(F8).view(*codes.shape[:-1], 64)
    return {"values": values, "groups": groups, "scales": scales, "q": q_out}


def _run_write(s):
    dim = s["k"].shape[-1]
    if own:
        _pkg().run_kv4_write(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"], s["slots"],
                             s["cache"], s["q_out"], eps=EPS, interleaved=s["interleaved"])
        return _write_outputs(s["cache"], dim, s["q_out"])
    turn = s["cos_sin"][s["positions"]]
    _put(s["cache"], 0, s["slots"], _rotated(_normed(s["k"].float(), s["k_weight"]), turn, s["interleaved"]))
    _put(s["cache"], 1, s["slots"], s["v"].float())
    s["q_out"].copy_(_rotated(_normed(s["q"].float(), s["q_weight"]), turn, s["interleaved"]))
    return _write_outputs(s["cache"], dim, s["q_out"])


def _dequantised(codes, groups, scales):
    """f32 [..., D] of codes [..., D / 64, 32] (bytes), groups [..., D / 16] and scales [...]."""
    x = _table("values")[torch.stack([codes & 15, codes >> 4], dim=-1).int()].flatten(-3)
    return (x.unflatten(-1, (-1, GROUP)) * (groups.float() * scales[..., None])[..., None]).flatten(-2)


def _run_read(s):
    if own:
        _pkg().run_kv4_read(s["cache"], s["slots"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    codes, groups, scales = _views(s["cache"], s["dim"])
    page, at = s["slots"].clamp_min(0) // PAGE, s["slots"].clamp_min(0) % PAGE
    rows = _dequantised(codes[page, :, :, :, at], groups.view(torch.uint8)[page, :, :, at].view(F8), scales[page, :, :, at])   # [n, 2, heads, D]
    rows = torch.where((s["slots"] >= 0)[:, None, None, None], rows, 0.0).to(torch.bfloat16)
    return rows[:, 0], rows[:, 1]


def _run_attention(s):
    q, window = s["q"], s["window"]
    if own:
        return _pkg().run_kv4_attention(q, s["cache"], s["table"], s["seq_lens"], s["q_starts"], s["out"], window=window)
    (T, HQ, D), HK = q.shape, s["cache"].shape[2]
    Q, G = s["longest_q"], HQ // HK
    n_q = s["q_starts"][1:] - s["q_starts"][:-1]
    codes, groups, scales = _views(s["cache"][s["table"]], D)
    kv = _dequantised(codes.transpose(-3, -2), groups, scales).permute(2, 0, 3, 1, 4, 5).flatten(3, 4)   # [2, B, heads, tokens, D]
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
    held = D // 2 + D // GROUP + 4          # bytes of a vector in the cache
    if case["op"] == "write":
        T, HQ, HK = case["tokens"], case["q_heads"], case["kv_heads"]
        kept = T - case["padded"]
        vectors = T * HQ + kept * 2 * HK
        size = vectors * D * 2 + T * (case["rotary"] * 4 + 8) + T * HQ * D * 2 + kept * 2 * HK * held
        return {"bytes": size, "flops": vectors * D * 8}
    if case["op"] == "read":
        rows, there = case["rows"] * case["kv_heads"] * 2, (case["rows"] - case["missing"]) * case["kv_heads"] * 2
        return {"bytes": there * held + rows * D * 2 + case["rows"] * 4, "flops": there * D}
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
    return {"bytes": sum(q_lens) * case["q_heads"] * D * 4 + read * case["kv_heads"] * 2 * held,
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


def _exact_codes(bytes_):
    """f64 [..., D] that bytes [..., D / 64, 32] stand for: sign, two bits of exponent, one of mantissa."""
    code = torch.stack([bytes_.long() % 16, bytes_.long() // 16], dim=-1).flatten(-3)
    exponent, mantissa = code // 2 % 4, (code % 2).double()
    value = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * torch.exp2(exponent.double() - 1))
    return torch.where(code >= 8, -value, value)


def _exact_write(s):
    """Scales and group scales before their rounding.  A code is a choice between two neighbours and has no such value."""
    dim = s["k"].shape[-1]
    turn = s["cos_sin"][s["positions"].long()]
    _, groups, scales = _views(s["cache"], dim)
    groups, scales = groups.double(), scales.double()
    written = [_exact_vectors(s["k"], s["k_weight"], turn, s["interleaved"]), _exact_vectors(s["v"], None, None, False)]
    slots = s["slots"].long()
    keep = slots >= 0
    page, at = slots[keep] // PAGE, slots[keep] % PAGE
    for kind, x in enumerate(written):
        largest = x[keep].abs().reshape(len(page), -1, dim // GROUP, GROUP).max(dim=-1).values
        scale = largest.max(dim=-1).values.clamp(min=1e-12) / 2688.0
        groups[page, kind, :, at] = largest / (6.0 * scale[..., None])
        scales[page, kind, :, at] = scale
    return {"values": None, "groups": groups, "scales": scales, "q": _exact_vectors(s["q"], s["q_weight"], turn, s["interleaved"])}


def _exact_tokens(s, slots, dim):
    """(keys, values) [n, heads, D] in 64 bits of cache rows."""
    codes, groups, scales = _views(s["cache"], dim)
    page, at = slots // PAGE, slots % PAGE
    groups = groups.view(torch.uint8)
    return [_exact_codes(codes[page, kind, :, :, at]) * groups[page, kind, :, at].view(F8).double().repeat_interleave(GROUP, dim=-1)
            * scales[page, kind, :, at].double()[..., None] for kind in range(2)]


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
