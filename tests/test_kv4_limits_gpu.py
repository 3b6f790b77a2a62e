"""Attention over the 4-bit cache where its numbers are at the ends of their ranges.  Tolerances are those of the definition's tests.  Needs a B200."""
import pytest
import torch

from test_kv4_gpu import _attend, _attention_inputs, _check_attention, kv4  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_len", [1, 40, 200])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("q_factor,key_factor,scale", [(1e-36, 1e38, None), (1e-35, 3e36, None), (1e-36, 3e37, -0.2), (1e-38, 1e38, 2.0)])
@pytest.mark.parametrize("D", [64, 128])
def test_tiny_queries_and_huge_keys(D, q_factor, key_factor, scale, window, q_len, pkg, kv4):  # noqa: F811
    """Scores of some tens and hundreds from queries near the smallest numbers and keys near the largest."""
    q, cache, table, lens, starts = _attention_inputs(kv4, [q_len, 3], [700, 500], 8, 2, D, seed=23)
    q *= q_factor
    kv4.views(cache)[2][:, 0] *= key_factor
    inputs = (q, cache, table, lens, starts)
    out = _attend(pkg, inputs, scale=scale, window=window)
    assert out.isfinite().all()
    _check_attention(out, *kv4.attention(*inputs, scale=scale, window=window))


@pytest.mark.parametrize("HQ,HK,D", [(4096, 1, 64), (4096, 1, 128), (1000, 2, 128), (514, 1, 64)])
@pytest.mark.parametrize("q_lens,kv_lens,window", [([1], [300], 0), ([2, 1], [150, 64], 0), ([3], [700], 100)])
def test_many_query_heads_to_a_key_head(q_lens, kv_lens, window, HQ, HK, D, pkg, kv4):  # noqa: F811
    """Up to the most there are: a token's heads are several row tiles."""
    inputs = _attention_inputs(kv4, q_lens, kv_lens, HQ, HK, D, seed=24)
    _check_attention(_attend(pkg, inputs, window=window), *kv4.attention(*inputs, window=window))


@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("HK", [1024, 300])
def test_many_key_heads(HK, q_len, pkg, kv4):  # noqa: F811
    inputs = _attention_inputs(kv4, [q_len, 2], [130, 65], HK, HK, 64, seed=25)
    _check_attention(_attend(pkg, inputs), *kv4.attention(*inputs))


@pytest.mark.parametrize("HQ,HK", [(4, 2), (40, 1)])
@pytest.mark.parametrize("every", [1, 3])
def test_the_largest_batch(every, HQ, HK, pkg, kv4):  # noqa: F811
    """65536 sequences, every one or every third of which has a token, of one position: results are the values themselves."""
    batch, D, pages = 1 << 16, 64, 50
    cache = kv4.random_cache(pages, HK, D, 4, "cuda:0")
    counts = (torch.arange(batch, device="cuda:0") % every == every - 1).int()
    table = (torch.arange(batch, device="cuda:0") % pages).to(torch.int32)[:, None]
    starts = torch.cat([counts.new_zeros(1), counts.cumsum(0).int()])
    q = torch.randn(int(starts[-1]), HQ, D, device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(1)).to(torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    pkg.run_kv4_attention(q, cache, table, torch.ones_like(counts), starts, out)
    pkg.kv4_check()
    want = kv4.rows(cache, table[counts > 0, 0] * 64, 1).repeat_interleave(HQ // HK, dim=1)
    assert ((out.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -11) * 1.01).all()       # the outputs' bf16, a weight's f16
