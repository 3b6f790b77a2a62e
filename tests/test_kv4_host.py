"""Host-side checks of the paged KV cache in 4 bits and the attention over it: no GPU needed."""
import ctypes
import math
import os
import re
from importlib import import_module

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCK = 64 * 76


def test_header_symbols_are_exported_and_bound(pkg):
    """Every function include/syfi_kv4.h declares is exported by the shared library and bound by the Python mirror."""
    text = open(os.path.join(ROOT, "include", "syfi_kv4.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\bint (syfi_[a-z0-9_]+)\s*\(", text)))
    assert "syfi_kv4_write" in names and "syfi_kv4_read" in names and "syfi_kv4_attention" in names
    lib = ctypes.CDLL(pkg.library_path())
    for n in names:
        assert hasattr(lib, n), f"{n} declared in include/syfi_kv4.h but not exported"
    assert sorted(import_module(pkg.__name__ + ".kv4").ABI.keys()) == names


def test_host_tensors_and_bad_shapes_are_refused(pkg):
    cache = torch.zeros(pkg.kv4_cache_shape(2, 1), dtype=torch.uint8)
    assert cache.shape == (2, 2, 1, BLOCK) and pkg.kv4_cache_shape(3, 5, 64) == (3, 2, 5, 64 * 40)
    with pytest.raises(ValueError, match="head_dim"):
        pkg.kv4_cache_shape(1, 1, 96)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.run_kv4_read(cache, torch.zeros(1, dtype=torch.int32), None, None)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.run_kv4_write(None, None, None, None, None, None, None, None, cache, None)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.run_kv4_attention(None, cache, None, None, None, None)


def _fn(pkg, name):
    import_module(pkg.__name__ + ".kv4")._lib()
    return getattr(pkg.load_library(), name)


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=96), "head_dim"), (dict(kv_heads=0), "kv_heads"), (dict(num_pages=0), "num_pages"), (dict(num_pages=1 << 25), "num_pages"),
    (dict(page_stride=2 * BLOCK - 16), "page_stride"), (dict(page_stride=2 * BLOCK + 8), "page_stride"), (dict(cache=8), "cache"), (dict(cache=None), "cache"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 40), "tokens"), (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=144), "rotary_dim"),
    (dict(max_positions=0), "cos_sin"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(q=None), "null"),
    (dict(q_out=4096 + 8), "aligned"), (dict(slots=2), "aligned"), (dict(cos_sin=None), "null"), (dict(k_stride=120), "stride"), (dict(v_stride=129), "stride"),
])
def test_write_checks_its_arguments_before_the_device(change, message, pkg):
    """Through the C ABI: bad arguments come back as code 1 with a message, on any machine."""
    p = 4096
    args = dict(q=p, k=p, v=p, q_weight=p, k_weight=p, cos_sin=p, positions=p, slots=p, tokens=4, q_heads=2, kv_heads=1, head_dim=128,
                rotary_dim=128, interleaved=0, max_positions=9, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, eps=1e-6,
                cache=p, num_pages=2, page_stride=2 * BLOCK, q_out=p, stream=None)
    args.update(change)
    assert _fn(pkg, "syfi_kv4_write")(*args.values()) == 1
    assert message in pkg.load_library().syfi_moe_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(head_dim=100), "head_dim"), (dict(rows=-1), "rows"), (dict(slots=None), "null"), (dict(k_out=4), "aligned"), (dict(cache=24), "cache"),
])
def test_read_checks_its_arguments_before_the_device(change, message, pkg):
    p = 4096
    args = dict(cache=p, num_pages=2, page_stride=2 * BLOCK, kv_heads=1, head_dim=128, slots=p, rows=4, out_f32=0, k_out=p, v_out=p, stream=None)
    args.update(change)
    assert _fn(pkg, "syfi_kv4_read")(*args.values()) == 1
    assert message in pkg.load_library().syfi_moe_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(q_heads=7, kv_heads=2), "multiple"), (dict(batch=-1), "batch"), (dict(tokens=1 << 40), "tokens"), (dict(max_pages=0), "max_pages"), (dict(window=-1), "window"),
    (dict(scale=math.inf), "scale"), (dict(q=None), "null"), (dict(out=4), "aligned"), (dict(q_starts=None), "null"), (dict(q_stride=64), "stride"),
    (dict(out_stride=260), "stride"), (dict(page_stride=1), "page_stride"),
])
def test_attention_checks_its_arguments_before_the_device(change, message, pkg):
    p = 4096
    args = dict(q=p, q_stride=256, cache=p, num_pages=9, page_stride=4 * BLOCK, block_table=p, max_pages=3, seq_lens=p, q_starts=p, batch=2, tokens=4, q_heads=2,
                kv_heads=2, head_dim=128, scale=1.0, window=0, out=p, out_stride=256, stream=None)
    args.update(change)
    assert _fn(pkg, "syfi_kv4_attention")(*args.values()) == 1
    assert message in pkg.load_library().syfi_moe_last_error().decode()


@pytest.mark.parametrize("name,index", [("syfi_kv4_attention", 15), ("syfi_kv4_attention", 11), ("syfi_kv4_attention", 6), ("syfi_kv4_write", 9), ("syfi_kv4_read", 3)])
@pytest.mark.parametrize("value", [2 ** 32 + 1, 2 ** 31, -2 ** 32 + 1])
def test_a_block_refuses_what_does_not_fit_in_32_bits(name, index, value, pkg):
    """A block's words are 64 bits wide, some of the arguments they stand for 32: no word is cut.  (No call here has any work.)"""
    p = 4096
    blocks = {"syfi_kv4_attention": [p, 256, p, 9, 4 * BLOCK, p, 3, p, p, 0, 0, 2, 2, 128, 1.0, 0, p, 256, 0],
              "syfi_kv4_write": [p, p, p, p, p, p, p, p, 0, 2, 1, 128, 128, 0, 9, 256, 128, 128, 256, 1e-6, p, 2, 2 * BLOCK, p, 0],
              "syfi_kv4_read": [p, 2, 2 * BLOCK, 1, 128, p, 0, 0, p, p, 0]}
    module = import_module(pkg.__name__ + ".kv4")
    call = _fn(pkg, name + "_block")
    assert call(module._block(name)(*blocks[name])) == 0
    args = list(blocks[name])
    args[index] = value
    assert call(module._block(name)(*args)) == 1
    assert "32 bits" in pkg.load_library().syfi_moe_last_error().decode()
    assert call(None) == 1


@pytest.mark.parametrize("tokens", [2 ** 61 + 1, 2 ** 62, 2 ** 63 - 1, (2 ** 31 - 1) // 8 + 1])
def test_write_refuses_tokens_whose_product_does_not_fit(tokens, pkg):
    p = 4096
    assert _fn(pkg, "syfi_kv4_write")(p, p, p, None, None, None, None, p, tokens, 6, 1, 128, 0, 0, 0, 768, 128, 128, 768, 1e-6, p, 2, 2 * BLOCK, p, None) == 1
    assert "tokens" in pkg.load_library().syfi_moe_last_error().decode()


def test_oracle_codes_and_layout():
    """Codes by hand, ties among them; a row put together byte by byte as the header says reads back as what it stands for."""
    kv4 = import_module("oracle.kv4_oracle")
    x = torch.tensor([0.0, 0.25, 0.250001, 0.75, 1.25, 1.26, 1.75, 2.5, 2.51, 3.5, 5.0, 5.1, 7.0, -0.2, -0.75, -6.5], dtype=torch.float64)
    assert kv4.nearest_codes(x).tolist() == [0, 0, 1, 2, 2, 3, 4, 4, 5, 6, 6, 7, 7, 8, 10, 15]
    for dim in (64, 128):
        cache = torch.zeros(2, 2, 3, 64 * (dim // 2 + dim // 16 + 4), dtype=torch.uint8)
        assert kv4.dim_of(cache) == dim
        g = torch.Generator().manual_seed(dim)
        z = torch.randn(3, dim, generator=g)
        codes, groups, scales = kv4.quantised(z)
        at = 37
        for h in range(3):
            block = cache[1, 1, h]
            for d in range(dim):
                block[d // 64 * 2048 + at * 32 + d % 64 // 2] |= int(codes[h, d]) << (4 * (d % 2))
            block[32 * dim + at * (dim // 16):][: dim // 16] = groups[h].to(kv4.F8).view(torch.uint8)
            block[36 * dim + 4 * at:][:4] = scales[h].float().view(1).view(torch.uint8)
        got = kv4.rows(cache, torch.tensor([64 + at, -1, 128]), 1)
        table = torch.tensor(kv4.VALUES, dtype=torch.float64)
        assert torch.equal(got[0], table[codes] * groups.repeat_interleave(16, dim=-1) * scales[:, None]) and (got[1:] == 0).all()
        # half of the step from 4 to 6 is a sixth of a group's largest; and the group scale's rounding
        top = z.abs().unflatten(-1, (-1, 16)).amax(-1).repeat_interleave(16, dim=-1)
        assert ((got[0] - z).abs() <= top * (1 / 6 + 2.0 ** -4)).all()


def test_oracle_against_a_dense_computation():
    """The oracle on one sequence whose pages lie in order equals a masked softmax over the dequantised rows."""
    kv4 = import_module("oracle.kv4_oracle")
    cache = kv4.random_cache(3, 2, 64, seed=1)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(5, 4, 64, generator=g).to(torch.bfloat16)
    out, spread, floor = kv4.attention(q, cache, torch.arange(3, dtype=torch.int32)[None], torch.tensor([150]), torch.tensor([0, 5]), window=20)
    keys, values = kv4.rows(cache, torch.arange(150), 0), kv4.rows(cache, torch.arange(150), 1)
    for i in range(5):
        p = 145 + i
        for h in range(4):
            w = torch.softmax(keys[p - 19: p + 1, h // 2] @ q[i, h].double() / 8, 0)
            assert torch.allclose(out[i, h], w @ values[p - 19: p + 1, h // 2], rtol=1e-12)
    assert (spread >= out.abs() - 1e-12).all() and (floor > 0).all() and (floor < spread * 1e-5).all()
