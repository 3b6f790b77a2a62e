"""The serving example against the definitions in 64 bits, step by step.  Needs a B200.

Tolerance: the output in bf16 is off by 2^-8 of itself at most, weights in f16 by 2^-11 each, twice that is allowed, in units of the
average of |value| under the weights."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_serving_example_matches_the_definitions():
    import importlib
    kv = importlib.import_module("oracle.kv_oracle")
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.run()
    device = got["cache"].device
    table = got["table"].to(device)
    # (written bytes of a step stay as they are, and no step sees later ones: the last cache serves all steps)
    for lens, counts, q, out in got["steps"]:
        starts = torch.tensor([0] + counts, dtype=torch.int32, device=device).cumsum(0).to(torch.int32)
        want, spread = kv.attention(q, got["cache"], table, torch.tensor(lens, dtype=torch.int32, device=device), starts)
        assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -8 * 1.01 + spread * (2.0 ** -10 + 2.0 ** -12)).all()
    assert [sum(c) for c in zip(*(counts for _, counts, _, _ in got["steps"]))] == [p + example.NEW_TOKENS for p in example.PROMPTS]
    picked = got["picked"]
    assert (picked >= 0).all() and len(set(picked.tolist())) == 2048
    assert torch.equal(got["values"], kv.rows(got["cache"], picked, 1).float().to(torch.bfloat16))
    assert torch.equal(got["keys"], kv.rows(got["cache"], picked, 0).float().to(torch.bfloat16))
