"""The quantised paged KV cache and the attention over it against their definitions in 64 bits.  Needs a B200.

Tolerances follow from the number formats: a result in bf16 is off by half a unit in its last place (2^-8 of its value at most), a byte
of the cache by half an e4m3 step (2^-4 of its value, 2^-10 scales near zero), f32 arithmetic on a head's up to 128 dimensions by
a few 1e-6 of the vector's largest; attention weights may be rounded to f16 (2^-11 of each), twice that is allowed, in units of
the average of |value| under the weights."""
import ctypes
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def kv():
    return importlib.import_module("oracle.kv_oracle")


# ------------------------------------------------------------------------------------------------- write
def _turn(rows, rotary):
    angle = torch.arange(rows, device=DEV).double()[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2, device=DEV).double() / rotary)
    return torch.cat([angle.cos(), angle.sin()], dim=-1).float()


def _write_inputs(kv, T, HQ, HK, D, rotary, norm, kinds=2, seed=0, layers=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    fused = (torch.randn(T, (HQ + kinds * HK) * D + 8, generator=g, device=DEV) * torch.logspace(-3, 3, T, device=DEV)[:, None]).to(torch.bfloat16)
    q = fused[:, : HQ * D].unflatten(-1, (HQ, D)) if HQ else None
    k = fused[:, HQ * D: (HQ + HK) * D].unflatten(-1, (HK, D))
    v = fused[:, (HQ + HK) * D: (HQ + 2 * HK) * D].unflatten(-1, (HK, D)) if kinds == 2 else None
    w = [(torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16) if norm else None for _ in range(2)]
    pages = T // 64 + 3
    slots = torch.randperm(pages * 64, generator=g, device=DEV)[:T].to(torch.int32)
    slots[::7] = -1
    positions = torch.randint(0, 5000, (T,), generator=g, device=DEV, dtype=torch.int32)
    cache = torch.stack([kv.random_cache(pages, kinds, HK, D, seed + i, DEV) for i in range(layers)], dim=1)[:, layers // 2]
    q_out = torch.empty(T, HQ, D, dtype=torch.bfloat16, device=DEV) if HQ else None
    return q, k, v, w[0] if HQ else None, w[1], _turn(5000, rotary) if rotary else None, positions, slots, cache, q_out


def _check_written(kv, cache, before, slots, kind, z):
    """Written rows stand for z within the format's rounding; everything else keeps its bytes."""
    values, scales = kv.views(cache)
    keep = slots >= 0
    page, at = slots[keep].long() // 64, slots[keep].long() % 64
    want = z[keep]
    scale = scales[page, kind, :, at].double()
    exact = want.abs().amax(-1).clamp(min=1e-12) / 448
    assert ((scale - exact).abs() <= 4e-6 * exact).all()
    got = values.view(torch.uint8)[page, kind, :, at].view(F8).double() * scale[..., None]
    limit = torch.maximum(want.abs() * 2.0 ** -4, scale[..., None] * 2.0 ** -10) * 1.001 + 4e-6 * want.abs().amax(-1, keepdim=True)
    assert ((got - want).abs() <= limit).all()
    old_values, old_scales = kv.views(before)
    same = torch.ones(cache.shape[0], 64, dtype=torch.bool, device=DEV)
    same[page, at] = False
    same = same[:, None].expand(-1, cache.shape[2], -1)
    assert torch.equal(values.view(torch.uint8)[:, kind][same], old_values.view(torch.uint8)[:, kind][same])
    assert torch.equal(scales[:, kind][same], old_scales[:, kind][same])


@pytest.mark.parametrize("T,HQ,HK,D,rotary,interleaved,norm,layers", [
    (1, 32, 8, 128, 128, False, True, 1),
    (1, 1, 1, 64, 64, True, True, 1),
    (63, 12, 4, 128, 64, False, True, 3),        # half of the dimensions turned; a layer's slice of a cache of three
    (65, 5, 5, 64, 16, False, False, 2),
    (130, 40, 8, 64, 48, True, True, 1),
    (257, 3, 1, 128, 96, False, True, 1),        # pairs 48 apart: partners that are no power of two of lanes away
    (1000, 24, 8, 128, 0, False, True, 1),       # no rotation
    (777, 7, 7, 128, 128, True, False, 1),
    (2500, 64, 1, 128, 128, False, True, 1),
])
def test_write_matches_the_definition(T, HQ, HK, D, rotary, interleaved, norm, layers, pkg, kv):
    q, k, v, qw, kw, turn, positions, slots, cache, q_out = _write_inputs(kv, T, HQ, HK, D, rotary, norm, layers=layers)
    before = cache.clone()
    assert pkg.run_kv_write(q, k, v, qw, kw, turn, positions if rotary else None, slots, cache, q_out, interleaved=interleaved) is q_out
    want = kv.head_vectors(q, qw, turn, positions, interleaved=interleaved)
    assert ((q_out.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.001 + 4e-6 * want.abs().amax(-1, keepdim=True)).all()
    _check_written(kv, cache, before, slots, 0, kv.head_vectors(k, kw, turn, positions, interleaved=interleaved))
    _check_written(kv, cache, before, slots, 1, v.double())


@pytest.mark.parametrize("T,HQ,HK,D,rotary,interleaved", [
    (3000, 40, 5, 64, 48, False), (3000, 40, 5, 64, 64, True), (3000, 24, 9, 128, 128, True), (2600, 35, 7, 128, 96, False), (5000, 16, 16, 64, 16, True)])
def test_write_of_many_tokens_matches_the_definition(T, HQ, HK, D, rotary, interleaved, pkg, kv):
    """Enough vectors that a group of lanes takes a run of four heads; numbers of heads that leave a rest of a run."""
    q, k, v, qw, kw, turn, positions, slots, cache, q_out = _write_inputs(kv, T, HQ, HK, D, rotary, True, seed=5)
    before = cache.clone()
    pkg.run_kv_write(q, k, v, qw, kw, turn, positions, slots, cache, q_out, interleaved=interleaved)
    want = kv.head_vectors(q, qw, turn, positions, interleaved=interleaved)
    assert ((q_out.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.001 + 4e-6 * want.abs().amax(-1, keepdim=True)).all()
    _check_written(kv, cache, before, slots, 0, kv.head_vectors(k, kw, turn, positions, interleaved=interleaved))
    _check_written(kv, cache, before, slots, 1, v.double())


@pytest.mark.parametrize("T,HK,D", [(70, 3, 128), (1, 8, 64), (4000, 8, 128), (9000, 5, 64)])
def test_written_bytes_are_the_rounded_quotients(T, HK, D, pkg, kv):
    """Without norm and rotation: the scale is the division by 448 rounded once, the bytes are the division by the scale, rounded to f32
    and then to e4m3.  (A quotient of f32 numbers rounded to 53 bits and then to 24 is the one rounded at once.)"""
    g = torch.Generator(device=DEV).manual_seed(T)
    k, v = ((torch.randn(T, HK, D, generator=g, device=DEV) * torch.exp2(torch.randint(-40, 40, (T, HK, 1), generator=g, device=DEV).float())).to(torch.bfloat16) for _ in range(2))
    steps = torch.arange(D, device=DEV)                     # half way between two e4m3 numbers, for a scale of 1
    k[0, 0] = torch.where(steps == 0, 448.0, (17.0 + 2.0 * (steps % 8)) * torch.exp2((steps % 11).float() - 8.0)).to(torch.bfloat16)
    v[0, 0] = 0.0
    cache = kv.random_cache(T // 64 + 1, 2, HK, D, 3, DEV)
    slots = torch.randperm(cache.shape[0] * 64, generator=g, device=DEV)[:T].to(torch.int32)
    pkg.run_kv_write(None, k, v, None, None, None, None, slots, cache, None)
    values, scales = kv.views(cache)
    page, at = slots.long() // 64, slots.long() % 64
    for kind, x in enumerate((k.double(), v.double())):
        scale = (x.abs().amax(-1).clamp(min=float(torch.tensor(1e-12))) / 448.0).float()
        assert torch.equal(scales[page, kind, :, at], scale)
        want = (x / scale.double()[..., None]).float().to(F8).view(torch.uint8)
        assert torch.equal(values.view(torch.uint8)[page, kind, :, at], want)


@pytest.mark.parametrize("T,HK,rotary", [(1, 1, 64), (300, 1, 64), (70, 3, 128)])
def test_write_of_keys_only(T, HK, rotary, pkg, kv):
    _, k, _, _, kw, turn, positions, slots, cache, _ = _write_inputs(kv, T, 0, HK, 128, rotary, True, kinds=1)
    before = cache.clone()
    pkg.run_kv_write(None, k, None, None, kw, turn, positions, slots, cache.view(torch.int8), None)
    _check_written(kv, cache, before, slots, 0, kv.head_vectors(k, kw, turn, positions))


def test_write_into_the_queries_own_place_and_with_large_eps(pkg, kv):
    q, k, v, qw, kw, turn, positions, slots, cache, q_out = _write_inputs(kv, 100, 8, 2, 128, 128, True)
    want = kv.head_vectors(q, qw, turn, positions, eps=10.0)
    pkg.run_kv_write(q, k, v, qw, kw, turn, positions, slots, cache, q, eps=10.0)
    assert ((q.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.001 + 4e-6 * want.abs().amax(-1, keepdim=True)).all()


def test_write_of_zeros_infinities_nans_and_unknown_places(pkg, kv):
    """Zero vectors have the smallest scale; a vector with a NaN or an infinity is NaN and touches no other; positions outside the
    table give NaN, slots outside the cache nothing."""
    q, k, v, _, _, turn, positions, slots, cache, q_out = _write_inputs(kv, 16, 2, 2, 128, 128, False)
    slots[:] = torch.arange(16, dtype=torch.int32, device=DEV)
    k[3, 0] = 0
    v[3, 1] = 0
    v[4, 0, 5] = float("inf")
    v[5, 1, 100] = float("nan")
    k[6, 0, 0] = float("-inf")
    positions[7], positions[8] = -1, 5000
    slots[9], slots[10] = cache.shape[0] * 64, -(2 ** 31)
    before = cache.clone()
    pkg.run_kv_write(q, k, v, None, None, turn, positions, slots, cache, q_out)
    at = torch.arange(16, dtype=torch.int32, device=DEV)
    keys, values = kv.rows(cache, at, 0), kv.rows(cache, at, 1)
    assert (keys[3, 0] == 0).all() and (values[3, 1] == 0).all()
    assert float(kv.views(cache)[1][0, 1, 1, 3]) == pytest.approx(1e-12 / 448, rel=1e-5)
    nan_keys, nan_values = [(6, 0), (7, 0), (7, 1), (8, 0), (8, 1)], [(4, 0), (5, 1)]
    for got, bad in ((keys, nan_keys), (values, nan_values)):
        expect = torch.zeros(16, 2, dtype=torch.bool, device=DEV)
        for t, h in bad:
            expect[t, h] = True
        assert torch.equal(got.isnan().all(-1), expect) and torch.equal(got.isnan().any(-1), expect)
    assert torch.equal(q_out.isnan().all(-1).all(-1), (at == 7) | (at == 8))
    for t in (9, 10):
        assert torch.equal(kv.rows(cache, at[t:t + 1], 0), kv.rows(before, at[t:t + 1], 0))


def test_written_index_keys_are_what_the_indexer_reads(pkg, kv):
    """A keys-only cache of one head is the indexer's: its choice equals the oracle's on the same bytes, and the chosen rows come
    back by their ids."""
    from oracle import dsa_oracle
    n = 5000
    _, k, _, _, kw, turn, _, slots, cache, _ = _write_inputs(kv, n, 0, 1, 128, 64, True, kinds=1, seed=3)
    g = torch.Generator(device=DEV).manual_seed(4)
    pages = torch.randperm(cache.shape[0], generator=g, device=DEV).to(torch.int32)
    j = torch.arange(n, device=DEV)
    slots = (pages[j // 64] * 64 + j % 64).to(torch.int32)
    pkg.run_kv_write(None, k, None, None, kw, turn, (j % 5000).to(torch.int32), slots, cache, None)
    index_cache = cache.view(torch.int8).view(-1, 64, 1, 132)
    q = torch.randn(1, 64, 128, generator=g, device=DEV).to(F8)
    weights = torch.randn(1, 64, generator=g, device=DEV) / 8
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    table = pages[None, : (n + 63) // 64].contiguous()
    picked = torch.empty(1, 2048, dtype=torch.int32, device=DEV)
    pkg.run_dsa_topk_indexer(q, index_cache, weights, lens, table, picked)
    want, scores = dsa_oracle.topk_indexer(q, index_cache, weights, lens, table)
    ok, stats = dsa_oracle.check_topk(picked, want, scores, lens.cpu(), table.cpu())
    assert ok, stats
    rows = torch.empty(2048, 1, 128, dtype=torch.float32, device=DEV)
    pkg.run_kv_read(cache, picked[0], rows, None)
    assert torch.equal(rows, kv.rows(cache, picked[0], 0).float())


# ------------------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("rows,H,D,dtype,layers", [(1, 1, 64, torch.bfloat16, 1), (3, 8, 128, torch.float32, 2), (2049, 5, 64, torch.float32, 1),
                                                   (4097, 8, 128, torch.bfloat16, 1), (700, 3, 128, torch.bfloat16, 3)])
def test_read_matches_the_definition(rows, H, D, dtype, layers, pkg, kv):
    """One product and one rounding: the very bits."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    pages = rows // 64 + 2
    cache = torch.stack([kv.random_cache(pages, 2, H, D, i, DEV) for i in range(layers)], dim=1)[:, layers // 2]
    slots = torch.randint(-20, pages * 64 + 20, (rows + 1,), generator=g, device=DEV, dtype=torch.int32)[1:]
    k, v = (torch.full((rows, H, D), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    assert pkg.run_kv_read(cache, slots, k, v) == (k, v)
    for got, kind in ((k, 0), (v, 1)):
        want = kv.rows(cache, slots, kind).float()          # (an e4m3 value times an f32 scale, rounded once)
        assert torch.equal(got, want.to(dtype))
    alone = torch.empty_like(v)
    pkg.run_kv_read(cache, slots, None, alone)
    assert torch.equal(alone, v)


@pytest.mark.parametrize("rows,H,D,dtype", [(8000, 3, 64, torch.bfloat16), (8000, 5, 128, torch.float32), (8001, 5, 64, torch.float32), (13000, 3, 128, torch.bfloat16)])
def test_read_of_many_rows_matches_the_definition(rows, H, D, dtype, pkg, kv):
    """Enough vectors that a group of lanes takes four; odd numbers of heads, so that a run of four has keys and values."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    cache = kv.random_cache(rows // 64 + 2, 2, H, D, 4, DEV)
    slots = torch.randint(-20, cache.shape[0] * 64 + 20, (rows,), generator=g, device=DEV, dtype=torch.int32)
    k, v = (torch.full((rows, H, D), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    pkg.run_kv_read(cache, slots, k, v)
    alone = torch.empty_like(v)
    pkg.run_kv_read(cache, slots, None, alone)
    for got, kind in ((k, 0), (v, 1), (alone, 1)):
        assert torch.equal(got, kv.rows(cache, slots, kind).float().to(dtype))


def test_cache_beyond_four_gigabytes(pkg, kv):
    """Pages whose bytes lie behind the 32-bit range, for all three operators."""
    pages, H, D = 70000, 4, 128
    small = kv.random_cache(6, 2, H, D, 1, DEV)
    cache = torch.zeros(pkg.kv_cache_shape(pages, H, D), dtype=torch.uint8, device=DEV)
    assert 64000 * cache.stride(0) > 2 ** 32
    far = [pages - 1, pages - 7, 65000, 3, 69999 - 64, 64000]
    cache[far] = small
    j = torch.arange(6 * 64, device=DEV)
    slots = (torch.tensor(far, device=DEV)[j // 64] * 64 + j % 64).to(torch.int32)
    k, v = (torch.empty(384, H, D, dtype=torch.float32, device=DEV) for _ in range(2))
    pkg.run_kv_read(cache, slots, k, v)
    assert torch.equal(k, kv.rows(small, j, 0).float()) and torch.equal(v, kv.rows(small, j, 1).float())
    starts = torch.tensor([0, 200], dtype=torch.int32, device=DEV)
    lens = torch.tensor([380], dtype=torch.int32, device=DEV)
    q = torch.randn(200, 8, D, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(torch.bfloat16)
    outs = [torch.empty_like(q) for _ in range(2)]
    pkg.run_paged_attention(q, cache, torch.tensor([far], dtype=torch.int32, device=DEV), lens, starts, outs[0])
    pkg.run_paged_attention(q, small, torch.arange(6, dtype=torch.int32, device=DEV)[None], lens, starts, outs[1])
    assert torch.equal(outs[0], outs[1])
    x = torch.randn(1, 2 * H, D, device=DEV).to(torch.bfloat16)
    at = torch.tensor([(pages - 1) * 64 + 63], dtype=torch.int32, device=DEV)
    pkg.run_kv_write(x[:, :H], x[:, :H], x[:, H:], None, None, None, None, at, cache, torch.empty(1, H, D, dtype=torch.bfloat16, device=DEV))
    got = kv.rows(cache[pages - 1:], torch.tensor([63], device=DEV), 1)
    assert ((got - x[:, H:].double()).abs() <= x[:, H:].double().abs().amax(-1, keepdim=True) * 2.0 ** -4).all()


# ------------------------------------------------------------------------------------------------- attention
def _attention_inputs(kv, q_lens, kv_lens, HQ, HK, D, seed=0, q_scale=1.5, spare=2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [(n + 63) // 64 for n in kv_lens]
    pages = sum(need) + 3
    cache = kv.random_cache(pages, 2, HK, D, seed, DEV)
    place = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(kv_lens), max(need) + spare), 2 ** 30, dtype=torch.int32, device=DEV)    # (never to be followed)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = place[at: at + n]
        at += n
    starts = torch.tensor([0] + q_lens, dtype=torch.int32, device=DEV).cumsum(0).to(torch.int32)
    q = (torch.randn(sum(q_lens), HQ, D, generator=g, device=DEV) * q_scale).to(torch.bfloat16)
    return q, cache, table, torch.tensor(kv_lens, dtype=torch.int32, device=DEV), starts


def _check_attention(out, want, spread):
    assert torch.equal(out.isnan(), want.isnan())
    error = (out.double() - want).abs()
    limit = want.abs() * 2.0 ** -8 * 1.01 + spread * (2.0 ** -10 + 2.0 ** -12) + 1e-30
    bad = ~((error <= limit) | want.isnan())
    assert not bad.any(), (int(bad.sum()), float((error / limit).nan_to_num(0.0).max()), bad.nonzero()[:4].tolist())


def _attend(pkg, inputs, **kw):
    out = torch.full_like(inputs[0], float("nan"))
    assert pkg.run_paged_attention(*inputs, out, **kw) is out
    return out


@pytest.mark.parametrize("kv_lens", [[1], [63], [64], [65], [700], [127, 128, 129], [1, 2, 3, 5000], [300] * 40, [33000, 9], [4097, 1, 16385]])
@pytest.mark.parametrize("HQ,HK,D", [(32, 8, 128), (16, 16, 64), (64, 1, 128), (12, 4, 64), (40, 2, 128)])
def test_decoding_matches_the_definition(kv_lens, HQ, HK, D, pkg, kv):
    inputs = _attention_inputs(kv, [1] * len(kv_lens), kv_lens, HQ, HK, D)
    _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))


@pytest.mark.parametrize("q_lens,kv_lens,window", [
    ([64], [64], 0), ([65], [65], 0), ([128], [128], 0), ([129], [300], 0), ([1], [1], 0), ([700], [700], 0), ([257], [2000], 0),
    ([33, 1, 130], [33, 900, 1000], 0), ([500, 1, 1, 1, 20], [5000, 1, 64, 3000, 20], 0), ([2, 3, 2, 3], [200, 100, 128, 64], 0),
    ([300], [1500], 1), ([300], [1500], 64), ([300], [1500], 100), ([700, 40], [700, 5000], 333), ([1, 1, 1], [40, 1000, 5000], 128),
    ([90, 0, 50, 0], [90, 700, 64, 0], 0), ([0, 1], [5, 5], 0), ([1025], [1025], 5000), ([2, 2], [20000, 129], 0),
])
@pytest.mark.parametrize("HQ,HK,D", [(32, 8, 128), (8, 8, 64), (64, 1, 128), (15, 3, 64)])
def test_chunks_match_the_definition(q_lens, kv_lens, window, HQ, HK, D, pkg, kv):
    inputs = _attention_inputs(kv, q_lens, kv_lens, HQ, HK, D, seed=1)
    _check_attention(_attend(pkg, inputs, window=window), *kv.attention(*inputs, window=window))


@pytest.mark.parametrize("batch", [128, 129, 300, 1000])
@pytest.mark.parametrize("new_tokens", ["one", "few", "chunk"])
@pytest.mark.parametrize("D", [64, 128])
def test_batches_of_many_sequences(batch, new_tokens, D, pkg, kv):
    """Ragged batches around and beyond 128 sequences, some without a new token; by the average of the rows per sequence that is either
    kernel's work."""
    pick = lambda b, n: (b * 7919 + 13) % n  # noqa: E731
    q_lens = [0 if pick(b, 11) == 0 else 1 if new_tokens == "one" else 1 + pick(b, 3) for b in range(batch)]
    if new_tokens == "chunk":
        q_lens[batch // 2], q_lens[-1] = 300, 7 * batch
    kv_lens = [n + pick(b, 2000 if b % 16 == 0 else 130) for b, n in enumerate(q_lens)]
    inputs = _attention_inputs(kv, q_lens, kv_lens, 8, 2, D, seed=9)
    _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [500, 130, 64]), ([40, 200], [600, 200])])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_seen_does_not_matter(q_lens, kv_lens, D, pkg, kv):
    """NaN bytes, NaN and infinite scales behind a sequence's end, in front of a window, at later positions and in absent pages
    leave every bit; a NaN that is seen makes its rows NaN and no others."""
    inputs = _attention_inputs(kv, q_lens, kv_lens, 16, 4, D, seed=2)
    q, cache, table, lens, starts = inputs
    clean = _attend(pkg, inputs, window=100)
    values, scales = kv.views(cache)
    for b, n in enumerate(kv_lens):
        page, at = int(table[b, (n - 1) // 64]), (n - 1) % 64 + 1
        values.view(torch.uint8)[page, :, :, at:] = 0x7f
        scales[page, :, :, at:] = float("inf")
        seen_from = n - q_lens[b] - 99
        for j in range(0, max(seen_from, 0)):
            values.view(torch.uint8)[int(table[b, j // 64]), :, :, j % 64] = 0xff
            scales[int(table[b, j // 64]), :, :, j % 64] = float("nan")
    assert torch.equal(_attend(pkg, inputs, window=100), clean)
    last = len(kv_lens) - 1                                  # the last sequence's last position: only its last query sees it
    n = kv_lens[last]
    scales[int(table[last, (n - 1) // 64]), 1, 2, (n - 1) % 64] = float("nan")
    poisoned = _attend(pkg, inputs, window=100)
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    hit[-1, 8:12] = True
    assert torch.equal(poisoned.isnan().all(-1), hit) and torch.equal(poisoned.isnan().any(-1), hit)
    assert torch.equal(poisoned[~hit], clean[~hit])


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1, 1], [400, 64, 5000, 65]), ([300, 64, 100], [1000, 64, 100])])
@pytest.mark.parametrize("HQ,HK,D", [(16, 4, 128), (8, 1, 64)])
def test_absent_pages_and_rows_that_see_nothing(q_lens, kv_lens, HQ, HK, D, pkg, kv):
    """Positions of negative entries are not there; a row whose every position is missing, or that lies in front of its sequence,
    is zero."""
    inputs = _attention_inputs(kv, q_lens, kv_lens, HQ, HK, D, seed=3)
    q, cache, table, lens, starts = inputs
    table[0, ::2] = -1
    table[1, :] = -7
    table[2, 1:3] = 2 ** 24
    want, spread = kv.attention(*inputs)
    out = _attend(pkg, inputs)
    _check_attention(out, want, spread)
    assert (out[starts[1]:starts[2]] == 0).all()
    lens[2] = q_lens[2] - 1 if q_lens[2] > 1 else 0          # fewer positions than new tokens
    out = _attend(pkg, inputs)
    _check_attention(out, *kv.attention(*inputs))
    assert (out[starts[2]] == 0).all()


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 2], [100, 64, 1]), ([300, 64, 100], [1000, 64, 60])])
@pytest.mark.parametrize("HQ,HK,D", [(16, 4, 128), (8, 1, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_query_that_is_not_finite_and_sees_nothing(q_lens, kv_lens, HQ, HK, D, bad, pkg, kv):
    """It gets zeros like any other; where it sees something its head is NaN; no other row is touched."""
    inputs = _attention_inputs(kv, q_lens, kv_lens, HQ, HK, D, seed=12)
    q, cache, table, lens, starts = inputs
    table[1, :] = -1
    clean = _attend(pkg, inputs)
    rows = [0, q_lens[0], q_lens[0] + q_lens[1] - 1, q_lens[0] + q_lens[1], sum(q_lens) - 1]
    for row in rows:
        q[row, 1, 7] = bad
    out = _attend(pkg, inputs)
    blind = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    blind[starts[1]:starts[2]] = True
    blind[starts[2]:starts[2] + max(q_lens[2] - kv_lens[2], 0)] = True
    hit = torch.zeros_like(blind)
    hit[rows, 1] = True
    hit &= ~blind
    assert (out[blind] == 0).all()
    assert out[hit].isnan().all()
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("q_len,kv_len", [(1, 3000), (300, 3000)])
def test_strides_scale_and_extremes(q_len, kv_len, pkg, kv):
    """Slices of fused rows and of a cache of several layers, another scale; scores far apart, one weight of nearly 1 and a long
    tail of tiny ones, and value scales from 1e-30 to 1e10."""
    q, cache, table, lens, starts = _attention_inputs(kv, [q_len], [kv_len], 8, 2, 128, seed=4)
    wide = torch.zeros(q_len, 24, 128, dtype=torch.bfloat16, device=DEV)
    wide[:, 8:16] = q
    layers = torch.stack([cache, cache.flip(0), cache], dim=1)
    layers[:, 1] = cache
    out = torch.full_like(wide, 3.0)
    pkg.run_paged_attention(wide[:, 8:16], layers[:, 1], table, lens, starts, out[:, 16:], scale=0.3)
    want, spread = kv.attention(q, cache, table, lens, starts, scale=0.3)
    _check_attention(out[:, 16:], want, spread)
    assert (out[:, :16] == 3.0).all()
    out = torch.empty_like(q)
    pkg.run_paged_attention(q, cache, table, lens, starts, out, scale=-2.0)
    _check_attention(out, *kv.attention(q, cache, table, lens, starts, scale=-2.0))
    values, scales = kv.views(cache)
    scales[:, 1] = 10.0 ** torch.linspace(-30, 10, scales[:, 1].numel(), device=DEV).view(scales[:, 1].shape)
    pkg.run_paged_attention(q, cache, table, lens, starts, out)
    _check_attention(out, *kv.attention(q, cache, table, lens, starts))
    scales[:, 1] = 0.0
    pkg.run_paged_attention(q, cache, table, lens, starts, out)
    assert (out == 0).all()


@pytest.mark.parametrize("q_len", [1, 200])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 100, 2 ** 40 + 1])
def test_windows_wider_than_any_sequence(q_len, window, pkg, kv):
    inputs = _attention_inputs(kv, [q_len], [700], 8, 2, 128, seed=17)
    assert torch.equal(_attend(pkg, inputs, window=window), _attend(pkg, inputs))


@pytest.mark.parametrize("q_len", [5, 200])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 20])
def test_wide_windows_over_sequences_shorter_than_their_new_tokens(q_len, window, pkg, kv):
    """The first queries' positions are negative."""
    inputs = _attention_inputs(kv, [q_len, 1], [q_len, 100], 8, 2, 128, seed=18)
    inputs[3][0] = q_len // 2
    _check_attention(_attend(pkg, inputs, window=window), *kv.attention(*inputs, window=window))


@pytest.mark.parametrize("q_len", [1, 200])
@pytest.mark.parametrize("q_factor,key_factor,scale", [(1e-32, 1e32, None), (1e-36, 1e20, 1e15), (1.0, 1e28, 1e-29), (1e25, 1e-25, None), (1.0, 1.0, 0.0)])
def test_queries_keys_and_scales_of_any_size(q_len, q_factor, key_factor, scale, pkg, kv):
    """Scores of ordinary size from factors that are not."""
    q, cache, table, lens, starts = _attention_inputs(kv, [q_len], [700], 8, 2, 128, seed=13)
    q *= q_factor
    kv.views(cache)[1][:, 0] *= key_factor
    inputs = (q, cache, table, lens, starts)
    _check_attention(_attend(pkg, inputs, scale=scale), *kv.attention(*inputs, scale=scale))


@pytest.mark.parametrize("q_len", [1, 200])
@pytest.mark.parametrize("spike", [0, 1000, 29999])
def test_one_large_weight_and_a_long_tail(q_len, spike, pkg, kv):
    """All positions but one have the same score, 17 octaves below the one: the tail's weights together are a quarter of it."""
    n = 30000
    q, cache, table, lens, starts = _attention_inputs(kv, [q_len], [n], 4, 1, 128, seed=5)
    values, scales = kv.views(cache)
    values[:, 0] = 0.0
    q[:] = 1.0
    at = min(spike, n - q_len)
    values[int(table[0, at // 64]), 0, 0, at % 64, 0] = 1.0
    scales[int(table[0, at // 64]), 0, 0, at % 64] = 17.0 * 0.6931471805599453 * 128 ** 0.5
    inputs = (q, cache, table, lens, starts)
    _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))


@pytest.mark.parametrize("q_len", [1, 2, 200])
@pytest.mark.parametrize("kv_len", [300, 9000])
@pytest.mark.parametrize("octaves", [60, 110, 150, 400])
def test_a_zero_value_far_above_the_others(q_len, kv_len, octaves, pkg, kv):
    """Positions with a value scale of zero whose scores lie far above all others, first, last or in between: next to nothing is left of
    the others, and no NaN.  Then scores far below zero with nothing but such values."""
    for spike in (0, kv_len // 2, kv_len - q_len):
        inputs = _attention_inputs(kv, [q_len], [kv_len], 8, 1, 128, seed=19)
        q, cache, table, lens, starts = inputs
        values, scales = kv.views(cache)
        page, at = int(table[0, spike // 64]), spike % 64
        values.view(torch.uint8)[page, 0, 0, at] = 0
        values.view(torch.uint8)[page, 0, 0, at, 0] = 0x38      # 1
        q[:, :, 0] = 1.0
        scales[page, 0, 0, at] = octaves * 0.6931471805599453 * 128 ** 0.5
        scales[page, 1, 0, at] = 0.0
        _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))
    values.view(torch.uint8)[:, 0] = 0
    values.view(torch.uint8)[:, 0, :, :, 0] = 0xb8              # -1
    scales[:, 0] = octaves * 0.6931471805599453 * 128 ** 0.5
    scales[:, 1] = 0.0
    assert (_attend(pkg, inputs) == 0).all()


@pytest.mark.parametrize("HQ,HK,D", [(8, 1, 128), (4, 1, 64), (16, 1, 128), (14, 1, 64)])
def test_a_long_sequence_in_more_parts_than_a_warp_has_lanes(HQ, HK, D, pkg, kv):
    inputs = _attention_inputs(kv, [1], [60000], HQ, HK, D, seed=6)
    _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))


@pytest.mark.parametrize("q_len", [31, 32, 33, 64, 65])
@pytest.mark.parametrize("kv_len", [120, 128, 129, 257, 400, 6000])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_around_a_tile_and_references_that_move(q_len, kv_len, D, pkg, kv):
    """128 rows of a key head and one token more or less, over even and odd numbers of tiles.  Along the sequence scores and the
    values' scales grow, so that references follow, or fall, or jump up and down."""
    inputs = _attention_inputs(kv, [q_len, 3], [kv_len, 3000], 8, 2, D, seed=7)
    q, cache, table, lens, starts = inputs
    _, scales = kv.views(cache)
    kept = scales.clone()
    j = torch.arange(kv_len, device=DEV)
    page, at = table[0, j // 64].long(), j % 64
    wave = torch.where(j // 128 % 3 == 1, 5.0, -5.0)
    for window in (0, 333):
        for octaves in (12.0 * j / kv_len - 6, 6 - 12.0 * j / kv_len, wave):
            scales.copy_(kept)
            scales[page, 1, :, at] *= torch.exp2(octaves)[:, None]
            scales[page, 0, :, at] *= torch.exp2(octaves / 4)[:, None]
            _check_attention(_attend(pkg, inputs, window=window), *kv.attention(*inputs, window=window))


@pytest.mark.parametrize("q_lens,kv_lens,D", [([300, 5], [3000, 9000], 128), ([6] * 9, [4000] * 9, 64)])
def test_bounded_waits_run_out(q_lens, kv_lens, D, pkg, kv):
    """A wait that runs out ends its call with a status; rows that were not computed are NaN, all others are what they are, and
    the next call is undisturbed."""
    inputs = _attention_inputs(kv, q_lens, kv_lens, 8, 2, D, seed=8)
    clean = _attend(pkg, inputs)
    lib = pkg.load_library()
    failed = 0
    for limit in (1, 1, 64, 200, 1000, 5000):
        assert lib.syfi_kv_debug_wait_limit(ctypes.c_int64(limit)) == 0
        out = _attend(pkg, inputs)
        try:
            pkg.kv_check()
            assert torch.equal(out, clean)
        except pkg.MoeError as err:
            assert "status 301" in str(err), str(err)
            failed += 1
            done = ~out.isnan().any(-1)
            assert torch.equal(out[done], clean[done]) and not bool(done.all())
        assert torch.equal(_attend(pkg, inputs), clean), limit
        pkg.kv_check()
    assert failed >= 1, failed


def _ms(f, calls=5):
    times = []
    for _ in range(calls + 1):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        f()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end))
    return min(times[1:])


@pytest.mark.parametrize("q_lens,kv_lens,D", [([3000], [3000], 128), ([300], [20000], 64), ([1, 80, 1, 200], [400, 3000, 9000, 5000], 128)])
def test_one_tiny_value_is_right_and_does_not_cost_much(q_lens, kv_lens, D, pkg, kv):
    """A value scale far below the others, which f16 does not hold beside them: only rows that it decides are computed again.  All rows of a
    unit were, and a call took 200 to 1000 times as long."""
    inputs = _attention_inputs(kv, q_lens, kv_lens, 32, 8, D, seed=15)
    q, cache, table, lens, starts = inputs
    plain = _ms(lambda: _attend(pkg, inputs))
    for b in range(len(kv_lens)):
        for position in (0, kv_lens[b] // 2):
            kv.views(cache)[1][int(table[b, position // 64]), 1, :, position % 64] *= 2.0 ** -30
    tiny = _ms(lambda: _attend(pkg, inputs))
    _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))
    assert tiny < 20.0 * plain, (tiny, plain)


@pytest.mark.parametrize("q_len,kv_len", [(300, 300), (300, 2000), (40, 2500), (2, 6000)])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_tiny_values_decide(q_len, kv_len, D, pkg, kv):
    """Value scales 30 octaves apart, position by position, and queries of every other head that look away from the large ones."""
    inputs = _attention_inputs(kv, [q_len, 30], [kv_len, 700], 16, 2, D, seed=16)
    q, cache, table, lens, starts = inputs
    _, scales = kv.views(cache)
    values, _ = kv.views(cache)
    large = torch.arange(64, device=DEV) % 7 == 3
    scales[:, 1, :, ~large] *= 2.0 ** -30
    values.view(torch.uint8)[:, 0, :, large] = 0
    values.view(torch.uint8)[:, 0, :, large, 0] = 0xb8       # -1
    scales[:, 0, :, large] = 60.0 * D ** 0.5            # a score of -60 for those heads
    q[:, :, 0] = 0.0
    q[:, ::2, 0] = 1.0
    _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))
    assert not _attend(pkg, inputs).isnan().any()


@pytest.mark.parametrize("q_lens,kv_lens,D", [([2500, 200], [2500, 3000], 128), ([3000], [5000], 64)])
def test_rows_that_are_computed_again_do_not_run_into_the_wait_limit(q_lens, kv_lens, D, pkg, kv):
    """All queries look away from the one large value, so that every row of every unit is computed again.  That is no reason to give up,
    though no tile is finished meanwhile: the limit is 2^18 clocks, a seventh of a millisecond."""
    inputs = _attention_inputs(kv, q_lens, kv_lens, 32, 8, D, seed=14)
    q, cache, table, lens, starts = inputs
    values, scales = kv.views(cache)
    first = table[:, 0].long()
    scales[:, 1] *= 2.0 ** -30
    scales[first, 1, :, 0] *= 2.0 ** 30
    values.view(torch.uint8)[first, 0, :, 0] = 0
    values.view(torch.uint8)[first, 0, :, 0, 0] = 0xb8       # -1
    scales[first, 0, :, 0] = 60.0 * D ** 0.5                 # a score of -60
    q[:, :, 0] = 1.0
    out = torch.full_like(q, 7.0)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    assert pkg.load_library().syfi_kv_debug_wait_limit(ctypes.c_int64(1 << 18)) == 0
    begin.record()
    pkg.run_paged_attention(*inputs, out)
    end.record()
    pkg.kv_check()
    assert begin.elapsed_time(end) > 1.0             # (else this tests nothing)
    _check_attention(out, *kv.attention(*inputs))


@pytest.mark.parametrize("q_lens,kv_lens", [([1] * 5, [900, 20000, 3, 64, 7000]), ([400, 3], [5000, 6000])])
def test_attention_is_repeatable_on_several_streams_and_in_graphs(q_lens, kv_lens, pkg, kv):
    """The same bits in a row of calls, on side streams at once, and in a replayed graph whose inputs change."""
    sets = [_attention_inputs(kv, q_lens, kv_lens, 32, 4, 128, seed=10 + i) for i in range(4)]
    want = [_attend(pkg, s) for s in sets]
    outs = [torch.empty_like(w) for w in want]
    side = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, stream, out in zip(sets, side, outs):
            with torch.cuda.stream(stream):
                pkg.run_paged_attention(*s, out)
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        assert torch.equal(w, out)
    static, out = [t.clone() for t in sets[0]], torch.empty_like(want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        pkg.run_paged_attention(*static, out)
    for s, w in list(zip(sets, want)) * 2:
        for dst, src in zip(static, s):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_write_attend_and_read_in_a_row(pkg, kv):
    """A prompt in two chunks and three decoded tokens through all three operators, against 64 bits from the rows read back."""
    HQ, HK, D, page_of = 16, 4, 128, [5, 2, 7, 0]
    cache = torch.zeros(pkg.kv_cache_shape(8, HK, D), dtype=torch.uint8, device=DEV)
    table = torch.tensor([page_of], dtype=torch.int32, device=DEV)
    turn = _turn(512, D)
    g = torch.Generator(device=DEV).manual_seed(6)
    done = 0
    for n in (100, 60, 1, 1, 1):
        fused = torch.randn(n, (HQ + 2 * HK) * D, generator=g, device=DEV).to(torch.bfloat16)
        q, k, v = (x.unflatten(-1, (-1, D)) for x in fused.split([HQ * D, HK * D, HK * D], dim=-1))
        positions = torch.arange(done, done + n, dtype=torch.int32, device=DEV)
        slots = table[0][(positions // 64).long()] * 64 + positions % 64
        q_out = torch.empty(n, HQ, D, dtype=torch.bfloat16, device=DEV)
        pkg.run_kv_write(q, k, v, None, None, turn, positions, slots, cache, q_out)
        done += n
        lens, starts = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([done], [0, n]))
        inputs = (q_out, cache, table, lens, starts)
        _check_attention(_attend(pkg, inputs), *kv.attention(*inputs))


# ------------------------------------------------------------------------------------------------- refusals
def test_refusals(pkg, kv):
    q, k, v, qw, kw, turn, positions, slots, cache, q_out = _write_inputs(kv, 20, 8, 2, 128, 128, True)
    write = lambda **kw_: pkg.run_kv_write(*[kw_.get(n, x) for n, x in dict(q=q, k=k, v=v, q_weight=qw, k_weight=kw, cos_sin=turn, positions=positions,  # noqa: E731
                                                                         slots=slots, kv_cache=cache, q_out=q_out).items()])
    for match, wrong in [("no CPU path", dict(kv_cache=cache.cpu())), ("dtype", dict(kv_cache=cache.float())), ("shape", dict(kv_cache=cache[..., :-64])),
                         ("contiguous", dict(kv_cache=cache.transpose(1, 2))), ("k has shape", dict(k=k[:, :1])), ("k has dtype", dict(k=k.float())),
                         ("v must be None", dict(v=None)), ("v has shape", dict(v=v[:5])), ("q_out must be", dict(q_out=None)), ("go with q", dict(q=None)),
                         ("q_weight has shape", dict(q_weight=qw[:64])), ("k_weight has dtype", dict(k_weight=kw.float())), ("columns", dict(cos_sin=turn[:, :8])),
                         ("cos_sin must be contiguous", dict(cos_sin=turn[:, :64])), ("positions must be a", dict(positions=None)), ("positions has dtype", dict(positions=positions.long())),
                         ("slots has shape", dict(slots=slots[:-1])), ("slots is on", dict(slots=slots.cpu())), ("aligned", dict(k_weight=torch.cat([kw, kw])[1:129]))]:
        with pytest.raises(ValueError, match=match):
            write(**wrong)
    rows = torch.empty(20, 2, 128, dtype=torch.bfloat16, device=DEV)
    for match, args in [("slots must be", (cache, None, rows, rows)), ("k_out has shape", (cache, slots, rows[:3], rows)), ("v_out has dtype", (cache, slots, rows, rows.float())),
                        ("bfloat16 or float32", (cache, slots, rows.half(), None)), ("keys only", (cache[:, :1].contiguous(), slots, rows, rows)), ("no CPU path", (cache.cpu(), slots, rows, rows))]:
        with pytest.raises(ValueError, match=match):
            pkg.run_kv_read(*args)
    q, cache, table, lens, starts = _attention_inputs(kv, [3], [70], 8, 2, 128)
    out = torch.empty_like(q)
    attend = lambda more={}, **kw_: pkg.run_paged_attention(*[kw_.get(n, x) for n, x in dict(q=q, kv_cache=cache, block_table=table, seq_lens=lens, q_starts=starts, out=out).items()], **more)  # noqa: E731
    for match, wrong in [("hold keys and values", dict(kv_cache=cache[:, :1].contiguous())), ("multiple of the cache's", dict(q=q[:, :7])), ("q has shape", dict(q=q[..., :64])), ("out has dtype", dict(out=out.float())),
                         ("out has shape", dict(out=out[:2])), ("block_table has dtype", dict(block_table=table.long())), ("seq_lens has shape", dict(seq_lens=starts)),
                         ("q_starts has shape", dict(q_starts=lens)), ("block_table must be a 2-D", dict(block_table=table[0])), ("window", dict(more=dict(window=-1))), ("finite", dict(more=dict(scale=float("nan")))),
                         ("multiple of 8", dict(q=torch.empty(3, 8 * 128 + 4, dtype=torch.bfloat16, device=DEV)[:, :1024].unflatten(-1, (8, 128))))]:
        with pytest.raises(ValueError, match=match):
            attend(**wrong)
    attend()
    assert pkg.run_paged_attention(q[:0], cache, table, lens, torch.zeros(2, dtype=torch.int32, device=DEV), out[:0]).shape == (0, 8, 128)
    assert pkg.run_kv_read(cache, slots[:0], rows[:0], None)[0].shape == (0, 2, 128)
