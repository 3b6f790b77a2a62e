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
