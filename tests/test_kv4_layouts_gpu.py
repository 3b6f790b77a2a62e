"""The three operators of the paged KV cache in 4 bits on caches that begin, and whose pages lie apart, at multiples of 16 bytes which are none of
32.  They must give the bits that they give on a cache of its own.  Needs a B200."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
LAYOUTS = [(16, 0), (0, 16), (16, 16), (48, 80)]       # bytes in front of the cache, and between two pages


@pytest.fixture(scope="module")
def kv4():
    return importlib.import_module("oracle.kv4_oracle")


def _carved(cache, offset, gap):
    """The same cache inside a larger buffer of bytes that are NaN as scales."""
    pages, page = len(cache), cache[0].numel()
    pool = torch.full((offset + pages * (page + gap),), 0xff, dtype=torch.uint8, device=DEV)
    carved = pool[offset:].as_strided(cache.shape, (page + gap, *cache.stride()[1:]))
    carved.copy_(cache)
    assert carved.data_ptr() % 32 == offset % 32 and carved.stride(0) % 32 == gap % 32
    return carved, pool


@pytest.mark.parametrize("offset,gap", LAYOUTS)
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [700, 64, 3000]), ([3, 5], [900, 130]), ([40, 1, 300], [400, 1000, 300])])
@pytest.mark.parametrize("HQ,HK,D", [(16, 4, 128), (8, 1, 64), (6, 3, 64)])
def test_attention(q_lens, kv_lens, HQ, HK, D, offset, gap, pkg, kv4):
    need = [(n + 63) // 64 for n in kv_lens]
    cache = kv4.random_cache(sum(need) + 2, HK, D, 5, DEV)
    place = torch.randperm(len(cache), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = place[sum(need[:b]):][:n]
    table = table.to(DEV)
    lens = torch.tensor(kv_lens, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0] + q_lens, dtype=torch.int32, device=DEV).cumsum(0).to(torch.int32)
    q = torch.randn(sum(q_lens), HQ, D, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(torch.bfloat16)
    want, out = torch.empty_like(q), torch.full_like(q, float("nan"))
    pkg.run_kv4_attention(q, cache, table, lens, starts, want)
    pkg.run_kv4_attention(q, _carved(cache, offset, gap)[0], table, lens, starts, out)
    pkg.kv4_check()
    assert not want.isnan().any() and torch.equal(out, want)


@pytest.mark.parametrize("offset,gap", LAYOUTS)
@pytest.mark.parametrize("T,D", [(70, 128), (70, 64), (4000, 128), (4000, 64)])
def test_write_and_read(T, D, offset, gap, pkg, kv4):
    HQ, HK = 8, 3
    cache = kv4.random_cache(T // 64 + 3, HK, D, 6, DEV)
    carved, pool = _carved(cache, offset, gap)
    before = pool.clone()
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (torch.randn(T, h, D, generator=g, device=DEV).to(torch.bfloat16) for h in (HQ, HK, HK))
    weight = torch.randn(D, generator=g, device=DEV).to(torch.bfloat16)
    angle = torch.rand(T, D // 2, generator=g, device=DEV)
    turn = torch.cat([angle.cos(), angle.sin()], dim=-1)
    positions = torch.arange(T, dtype=torch.int32, device=DEV)
    slots = torch.randperm(len(cache) * 64, generator=g, device=DEV)[:T].to(torch.int32)
    outs = [torch.empty_like(q) for _ in range(2)]
    for into, out in zip((cache, carved), outs):
        pkg.run_kv4_write(q, k, v, weight, weight, turn, positions, slots, into, out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(cache, carved)
    between = torch.ones_like(pool, dtype=torch.bool)
    between[offset:].as_strided(carved.shape, carved.stride()).fill_(False)
    assert torch.equal(pool[between], before[between])          # what lies around the pages is as it was
    for dtype in (torch.bfloat16, torch.float32):
        rows = [torch.empty(T, HK, D, dtype=dtype, device=DEV) for _ in range(4)]
        pkg.run_kv4_read(cache, slots, rows[0], rows[1])
        pkg.run_kv4_read(carved, slots, rows[2], rows[3])
        assert torch.equal(rows[0], rows[2]) and torch.equal(rows[1], rows[3])
        assert torch.equal(rows[2], kv4.rows(carved, slots, 0).float().to(dtype))
