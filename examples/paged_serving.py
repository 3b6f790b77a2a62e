"""One attention layer of a serving loop over the quantised paged KV cache.

Three sequences share one cache.  Each step takes up to CHUNK tokens of every prompt that is not through and one token of every
sequence that is being decoded, in one batch: write the new keys and values, attend.  A keys-only cache of one head beside it is
what the DSA indexer reads; at the end the indexer picks 2048 tokens of the longest sequence and their rows are read back.

    python examples/paged_serving.py
"""
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pkg = importlib.import_module("mlsys-contest-syfi-agent-assisted_b200")

Q_HEADS, KV_HEADS, DIM, PAGE, CHUNK = 32, 8, 128, 64, 512
PROMPTS, NEW_TOKENS = (700, 130, 2500), 6


def rotation(positions, dim, device):
    angle = torch.arange(positions, device=device)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, device=device) / dim)
    return torch.cat([angle.cos(), angle.sin()], dim=-1).float()


class Pages:
    """Pages of the cache by sequence, taken from a free list as sequences grow."""

    def __init__(self, count, batch, most, device):
        self.free = list(range(count))[::-1]
        self.table = torch.full((batch, most), -1, dtype=torch.int32)
        self.device = device

    def slots(self, b, first, count):
        """Slots of `count` new tokens of sequence b from position `first` on."""
        for page in range((first + PAGE - 1) // PAGE, (first + count + PAGE - 1) // PAGE):
            self.table[b, page] = self.free.pop()
        j = torch.arange(first, first + count)
        return self.table[b, j // PAGE] * PAGE + j % PAGE


def run(device="cuda:0", seed=0):
    """Returns each step's (lens, counts, q, out), the caches, the page table and what was picked."""
    g = torch.Generator(device=device).manual_seed(seed)
    batch, longest = len(PROMPTS), max(PROMPTS) + NEW_TOKENS
    pages = Pages(sum((n + NEW_TOKENS) // PAGE + 1 for n in PROMPTS), batch, longest // PAGE + 1, device)
    count = len(pages.free)
    cache = torch.zeros(pkg.kv_cache_shape(count, KV_HEADS, DIM), dtype=torch.uint8, device=device)
    index_cache = torch.zeros(pkg.kv_cache_shape(count, 1, DIM, keys_only=True), dtype=torch.uint8, device=device)
    turn, half_turn = rotation(longest, DIM, device), rotation(longest, DIM // 2, device)
    q_weight, k_weight = (torch.ones(DIM, dtype=torch.bfloat16, device=device) for _ in range(2))
    done, steps = [0] * batch, []
    while any(n < p + NEW_TOKENS for n, p in zip(done, PROMPTS)):
        counts = [min(CHUNK, p - n) if n < p else int(n < p + NEW_TOKENS) for n, p in zip(done, PROMPTS)]
        positions = torch.cat([torch.arange(n, n + c) for n, c in zip(done, counts)]).to(torch.int32)
        slots = torch.cat([pages.slots(b, n, c) for b, (n, c) in enumerate(zip(done, counts))]).to(torch.int32)
        done = [n + c for n, c in zip(done, counts)]
        positions, slots, table = positions.to(device), slots.to(device), pages.table.to(device)
        lens = torch.tensor(done, dtype=torch.int32, device=device)
        starts = torch.tensor([0] + counts, dtype=torch.int32, device=device).cumsum(0).to(torch.int32)
        # what a model's fused projections would give: q, k, v side by side, and the index key
        fused = torch.randn(len(slots), (Q_HEADS + 2 * KV_HEADS) * DIM, generator=g, device=device).to(torch.bfloat16)
        q, k, v = (x.unflatten(-1, (-1, DIM)) for x in fused.split([Q_HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], dim=-1))
        index_key = torch.randn(len(slots), 1, DIM, generator=g, device=device).to(torch.bfloat16)
        rotated = torch.empty(len(slots), Q_HEADS, DIM, dtype=torch.bfloat16, device=device)
        out = torch.empty_like(rotated)
        pkg.run_kv_write(q, k, v, q_weight, k_weight, turn, positions, slots, cache, rotated)
        pkg.run_kv_write(None, index_key, None, None, None, half_turn, positions, slots, index_cache, None)
        pkg.run_paged_attention(rotated, cache, table, lens, starts, out)
        steps.append((list(done), counts, rotated, out))
    # the indexer's choice among the longest sequence's tokens, and their keys and values for a kernel that wants bf16
    b = max(range(batch), key=lambda i: done[i])
    table = pages.table[b:b + 1].to(device)
    index_q = torch.randn(1, 64, DIM, generator=g, device=device).to(torch.float8_e4m3fn)
    weights = torch.randn(1, 64, generator=g, device=device) / 8
    picked = torch.empty(1, 2048, dtype=torch.int32, device=device)
    pkg.run_dsa_topk_indexer(index_q, index_cache.view(torch.int8).view(-1, PAGE, 1, DIM + 4), weights, lens[b:b + 1].clone(), table, picked)
    keys, values = (torch.empty(2048, KV_HEADS, DIM, dtype=torch.bfloat16, device=device) for _ in range(2))
    pkg.run_kv_read(cache, picked[0], keys, values)
    pkg.kv_check()
    return {"steps": steps, "cache": cache, "index_cache": index_cache, "table": pages.table, "picked": picked[0], "keys": keys, "values": values}


if __name__ == "__main__":
    result = run()
    for lens, counts, _, out in result["steps"]:
        print("lengths", lens, "new tokens", counts, "mean |out| %.4f" % float(out.float().abs().mean()))
    print("picked", int((result["picked"] >= 0).sum()), "tokens; mean |value| %.4f" % float(result["values"].float().abs().mean()))
