"""Python mirror of the quantised paged KV cache and the attention over it (csrc/kv_cache.cu, csrc/paged_attention.cu behind the
C ABI of include/syfi_kv.h).

The cache is a uint8 or int8 tensor ``[pages, kinds, kv_heads, 64 * (head_dim + 4)]`` (:func:`kv_cache_shape`): blocks of 64
tokens of e4m3 bytes, then the tokens' f32 scales.  ``kinds`` is 2 (keys, values) or 1 (keys only).  Pages may lie apart (a layer's
slice ``cache[:, layer]`` of a cache of all layers); the rest of a page is contiguous.  A keys-only cache of one head of 128 is, as
``cache.view(torch.int8).view(pages, 64, 1, 132)``, the one that :func:`run_dsa_topk_indexer` reads.

Destination-passing like the rest of the package: calls enqueue on the current CUDA stream, do not synchronise and can be
captured in a CUDA graph.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from .moe import _check, _stream_ptr, load_library

PAGE = 64
_vp, _i32, _i64, _f64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_double
# name -> (restype, argtypes); must list every symbol include/syfi_kv.h declares
ABI = {
    "syfi_kv_write": (ctypes.c_int, [_vp] * 8 + [_i64] + [_i32] * 5 + [_i64] * 5 + [_f64, _vp, _i64, _i64, _i32, _vp, _vp]),
    "syfi_kv_read": (ctypes.c_int, [_vp, _i64, _i64, _i32, _i32, _i32, _vp, _i64, _i32, _vp, _vp, _vp]),
    "syfi_paged_attention": (ctypes.c_int, [_vp, _i64, _vp, _i64, _i64, _vp, _i32, _vp, _vp, _i32, _i64, _i32, _i32, _i32, _f64,
                                            _i32, _vp, _i64, _vp]),
    "syfi_kv_write_block": (ctypes.c_int, [ctypes.c_char_p]),
    "syfi_kv_read_block": (ctypes.c_int, [ctypes.c_char_p]),
    "syfi_paged_attention_block": (ctypes.c_int, [ctypes.c_char_p]),
    "syfi_kv_check": (ctypes.c_int, [_vp]),
}


def _block(name):
    """Packs a call's arguments into one block (ctypes takes 0.15 us for each argument, a block half a microsecond for all)."""
    return struct.Struct("=" + "".join("d" if t is _f64 else "q" for t in ABI[name][1])).pack


_pack_write, _pack_read, _pack_attention = (_block(n) for n in ("syfi_kv_write", "syfi_kv_read", "syfi_paged_attention"))
_bound = None      # the library once these functions are declared
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _lib():
    global _bound
    if _bound:
        return _bound
    lib = load_library()
    for name, (res, args) in ABI.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _bound = lib
    return lib


_bf16, _f32, _int, _u8, _i8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8, torch.int8


def kv_cache_shape(num_pages: int, kv_heads: int, head_dim: int = 128, keys_only: bool = False):
    """Shape of the uint8 tensor that holds ``num_pages`` pages of 64 tokens."""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    return (int(num_pages), 1 if keys_only else 2, int(kv_heads), PAGE * (head_dim + 4))


def _cache_of(t):
    """(pages, page stride in bytes, kinds, heads, head_dim) of a cache tensor."""
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError("kv_cache must be a CUDA tensor: this library has no CPU path")
    if t.dtype is not _u8 and t.dtype is not _i8:
        raise ValueError(f"kv_cache has dtype {t.dtype}, expected uint8 or int8")
    shape = t.shape
    if len(shape) != 4 or shape[1] not in (1, 2) or shape[3] not in (PAGE * 68, PAGE * 132):
        raise ValueError(f"kv_cache has shape {tuple(shape)}, expected [pages, 1 or 2, kv_heads, 64 * (head_dim + 4)] with head_dim 64 or 128")
    pages, kinds, heads, block = shape
    stride = t.stride()
    if stride[3] != 1 or (heads > 1 and stride[2] != block) or (kinds > 1 and stride[1] != heads * block):
        raise ValueError("the blocks of a page of kv_cache must be contiguous")
    return pages, stride[0] if pages > 1 else kinds * heads * block, kinds, heads, block // PAGE - 4


def _tokens_of(t, name, tokens, heads, dim, dev, dtype=_bf16):
    """Token stride of a [tokens, heads, dim] tensor whose heads lie side by side."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.shape != (tokens, heads, dim):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {(tokens, heads, dim)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    stride = t.stride()
    if stride[2] != 1 or (heads > 1 and stride[1] != dim):
        raise ValueError(f"the heads of a token of {name} must be contiguous")
    return stride[0] if tokens > 1 else heads * dim


def _expect(t, name, dtype, shape, dev):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _call(fn, device, args):
    if device == _current_device():
        rc = fn(args)
    else:
        with torch.cuda.device(device):
            rc = fn(args)
    if rc:
        _check(rc)


# Each entry point first looks at its arguments in one flat expression: on a decode step the kernels take a few microseconds, checks one
# by one with a message each take longer.  Whatever is not as it is in the ordinary case goes through those.
def _plain_cache(t):
    """(device, pages, page stride, kinds, heads, head_dim) of a cache as it is in the ordinary case, else None."""
    pages, kinds, heads, block = t.shape
    page_stride, kind_stride, head_stride, one = t.stride()
    dim = block // PAGE - 4
    device = t.get_device()
    if (device >= 0 and (t.dtype is _u8 or t.dtype is _i8) and (dim == 128 or dim == 64) and block == PAGE * (dim + 4) and pages > 1 and one == 1
            and head_stride == block and (kind_stride == heads * block or kinds == 1) and 1 <= kinds <= 2):
        return device, pages, page_stride, kinds, heads, dim
    return None


def _window_of(window):
    """As 32 bits: a window of 2^31 - 1 positions is as wide as any."""
    window = int(window)
    if window < 0:
        raise ValueError("window must not be negative")
    return window if window < 2 ** 31 else 2 ** 31 - 1


def _stream_of(stream, device):
    return _raw_stream(device) if stream is None and _raw_stream is not None else _stream_ptr(stream, device)


def run_kv_write(q, k, v, q_weight, k_weight, cos_sin, positions, slots, kv_cache, q_out, *, eps=1e-6, interleaved=False, stream=None):
    """New tokens' queries, keys and values in one pass: RMS norm of every head (``q_weight`` / ``k_weight`` bf16 [head_dim], or
    None), rotation by ``cos_sin[positions]`` (f32 [max_positions, rotary_dim]: cosines, then sines; or None), then ``q_out`` in
    bf16 and keys and values quantised to e4m3 by token and head into ``kv_cache`` at ``slots`` (int32 [tokens], page * 64 + offset,
    -1 = not written).  ``q``, ``k``, ``v`` are bf16 [tokens, heads, head_dim], possibly slices of a fused projection; ``q`` and
    ``q_out`` may both be None, ``v`` is None for a keys-only cache; ``q_out`` may be ``q``.  Returns ``q_out``."""
    try:
        device, pages, page_stride, kinds, heads, dim = _plain_cache(kv_cache)
        tokens, q_heads, rows, rotary = len(k), 0, 0, 0
        q_ptr = q_stride = q_out_ptr = q_out_stride = v_ptr = v_stride = qw_ptr = kw_ptr = turn_ptr = pos_ptr = 0
        k_stride, k1, k2 = k.stride()
        ok = (k.shape == (tokens, heads, dim) and k1 == dim and k2 == 1 and k.dtype is _bf16 and k.get_device() == device and tokens > 0
              and k_stride >= heads * dim and k_stride % 8 == 0
              and slots.shape == (tokens,) and slots.dtype is _int and slots.is_contiguous() and slots.get_device() == device
              and (v is None) == (kinds == 1))
        if ok and v is not None:
            v_stride, v1, v2 = v.stride()
            v_ptr = v.data_ptr()
            ok = v.shape == k.shape and v1 == dim and v2 == 1 and v.dtype is _bf16 and v.get_device() == device and v_stride >= heads * dim and v_stride % 8 == 0
        if ok and q is not None:
            q_heads = q.shape[1]
            (q_stride, q1, q2), (q_out_stride, o1, o2) = q.stride(), q_out.stride()
            q_ptr, q_out_ptr = q.data_ptr(), q_out.data_ptr()
            ok = (q.shape == (tokens, q_heads, dim) and q_out.shape == q.shape and q1 == dim and o1 == dim and q2 == 1 and o2 == 1 and q.dtype is _bf16
                  and q_out.dtype is _bf16 and q.get_device() == device and q_out.get_device() == device and q_stride >= q_heads * dim
                  and q_out_stride >= q_heads * dim and q_stride % 8 == 0 and q_out_stride % 8 == 0)
        elif q_out is not None or q_weight is not None:
            ok = False
        if ok and q_weight is not None:
            qw_ptr = q_weight.data_ptr()
            ok = q_weight.shape == (dim,) and q_weight.dtype is _bf16 and q_weight.is_contiguous() and q_weight.get_device() == device
        if ok and k_weight is not None:
            kw_ptr = k_weight.data_ptr()
            ok = k_weight.shape == (dim,) and k_weight.dtype is _bf16 and k_weight.is_contiguous() and k_weight.get_device() == device
        if ok and cos_sin is not None:
            rows, rotary = cos_sin.shape
            turn_ptr, pos_ptr = cos_sin.data_ptr(), positions.data_ptr()
            ok = (cos_sin.dtype is _f32 and cos_sin.is_contiguous() and cos_sin.get_device() == device and 0 < rotary <= dim and rotary % 16 == 0
                  and positions.shape == (tokens,) and positions.dtype is _int and positions.is_contiguous() and positions.get_device() == device)
    except (AttributeError, TypeError, ValueError, IndexError):
        ok = False
    if ok:
        _call(_lib().syfi_kv_write_block, device,
              _pack_write(q_ptr, k.data_ptr(), v_ptr, qw_ptr, kw_ptr, turn_ptr, pos_ptr, slots.data_ptr(), tokens, q_heads, heads, dim, rotary,
                          1 if interleaved else 0, rows, q_stride, k_stride, v_stride, q_out_stride, eps, kv_cache.data_ptr(), pages, page_stride,
                          kinds, q_out_ptr, _stream_of(stream, device)))
        return q_out
    pages, page_stride, kinds, heads, dim = _cache_of(kv_cache)
    dev = kv_cache.device
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("k must be a 3-D tensor [tokens, kv_heads, head_dim]")
    tokens = k.shape[0]
    k_stride = _tokens_of(k, "k", tokens, heads, dim, dev)
    if (v is None) != (kinds == 1):
        raise ValueError("v must be None exactly where the cache holds keys only")
    v_ptr = v_stride = q_ptr = q_stride = q_out_ptr = q_out_stride = q_heads = 0
    if v is not None:
        v_stride = _tokens_of(v, "v", tokens, heads, dim, dev)
        v_ptr = v.data_ptr()
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must be a 3-D tensor [tokens, q_heads, head_dim]")
        q_heads = q.shape[1]
        q_stride = _tokens_of(q, "q", tokens, q_heads, dim, dev)
        q_out_stride = _tokens_of(q_out, "q_out", tokens, q_heads, dim, dev)
        q_ptr, q_out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None or q_weight is not None:
        raise ValueError("q_out and q_weight go with q")
    qw_ptr = 0 if q_weight is None else _expect(q_weight, "q_weight", _bf16, (dim,), dev)
    kw_ptr = 0 if k_weight is None else _expect(k_weight, "k_weight", _bf16, (dim,), dev)
    rotary = rows = turn_ptr = pos_ptr = 0
    if cos_sin is not None:
        if not isinstance(cos_sin, torch.Tensor) or cos_sin.dim() != 2:
            raise ValueError("cos_sin must be a 2-D tensor [max_positions, rotary_dim]")
        rows, rotary = cos_sin.shape
        if rotary == 0 or rotary > dim or rotary % 16:
            raise ValueError(f"cos_sin has {rotary} columns, expected a multiple of 16 up to head_dim {dim}")
        turn_ptr = _expect(cos_sin, "cos_sin", _f32, (rows, rotary), dev)
        pos_ptr = _expect(positions, "positions", _int, (tokens,), dev)
    slots_ptr = _expect(slots, "slots", _int, (tokens,), dev)
    if tokens == 0:
        return q_out
    _call(_lib().syfi_kv_write_block, dev.index,
          _pack_write(q_ptr, k.data_ptr(), v_ptr, qw_ptr, kw_ptr, turn_ptr, pos_ptr, slots_ptr, tokens, q_heads, heads, dim, rotary,
                      1 if interleaved else 0, rows, q_stride, k_stride, v_stride, q_out_stride, eps, kv_cache.data_ptr(), pages,
                      page_stride, kinds, q_out_ptr, _stream_ptr(stream, dev.index)))
    return q_out


def run_kv_read(kv_cache, slots, k_out, v_out, *, stream=None):
    """Rows of the cache by slot (int32 [rows], -1 = not there: zeros; a sequence's indexer result is such a list): ``k_out`` and
    ``v_out`` [rows, kv_heads, head_dim], bf16 or both f32, get the dequantised keys and values; either may be None."""
    try:
        device, pages, page_stride, kinds, heads, dim = _plain_cache(kv_cache)
        rows, dtype = len(slots), k_out.dtype
        shape = (rows, heads, dim)
        ok = (slots.dtype is _int and slots.dim() == 1 and slots.is_contiguous() and slots.get_device() == device and rows > 0
              and (dtype is _bf16 or dtype is _f32) and k_out.shape == shape and k_out.is_contiguous() and k_out.get_device() == device
              and kinds == 2 and v_out.dtype is dtype and v_out.shape == shape and v_out.is_contiguous() and v_out.get_device() == device)
    except (AttributeError, TypeError, ValueError, IndexError):
        ok = False
    if ok:
        _call(_lib().syfi_kv_read_block, device,
              _pack_read(kv_cache.data_ptr(), pages, page_stride, kinds, heads, dim, slots.data_ptr(), rows, 1 if dtype is _f32 else 0,
                         k_out.data_ptr(), v_out.data_ptr(), _stream_of(stream, device)))
        return k_out, v_out
    pages, page_stride, kinds, heads, dim = _cache_of(kv_cache)
    dev = kv_cache.device
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
        raise ValueError("slots must be a 1-D tensor")
    rows = slots.shape[0]
    slots_ptr = _expect(slots, "slots", _int, (rows,), dev)
    if v_out is not None and kinds == 1:
        raise ValueError("v_out must be None: this cache holds keys only")
    dtype = None
    ptrs = []
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None and dtype is None:
            dtype = getattr(t, "dtype", None)
            if dtype is not _bf16 and dtype is not _f32:
                raise ValueError(f"{name} must be a bfloat16 or float32 tensor")
        ptrs.append(0 if t is None else _expect(t, name, dtype, (rows, heads, dim), dev))
    if rows and dtype is not None:
        _call(_lib().syfi_kv_read_block, dev.index,
              _pack_read(kv_cache.data_ptr(), pages, page_stride, kinds, heads, dim, slots_ptr, rows, 1 if dtype is _f32 else 0, ptrs[0], ptrs[1],
                         _stream_ptr(stream, dev.index)))
    return k_out, v_out


def run_paged_attention(q, kv_cache, block_table, seq_lens, q_starts, out, *, scale=None, window=0, stream=None):
    """Softmax attention of new tokens over the cache, their own keys and values (already written) included.

    ``q`` and ``out``: bf16 [tokens, q_heads, head_dim]; rows ``q_starts[b] .. q_starts[b + 1] - 1`` (int32 [batch + 1]) are the last
    positions of sequence b, which has ``seq_lens[b]`` (int32 [batch]) positions in the pages ``block_table[b]`` (int32
    [batch, max_pages]; a negative entry's 64 positions are not there).  A query sees its own position and those before it, with
    ``window`` > 0 only the last ``window`` of them; one that sees nothing gets zeros.  ``scale`` defaults to head_dim ** -0.5."""
    try:
        device, pages, page_stride, kinds, heads, dim = _plain_cache(kv_cache)
        tokens, q_heads, q_dim = q.shape
        (q_stride, q1, q2), (out_stride, o1, o2) = q.stride(), out.stride()
        batch, max_pages = block_table.shape
        ok = (kinds == 2 and q_dim == dim and q1 == dim and o1 == dim and q2 == 1 and o2 == 1 and q.dtype is _bf16 and out.dtype is _bf16
              and out.shape == q.shape and q.get_device() == device and out.get_device() == device and tokens > 0 and q_heads % heads == 0
              and q_stride >= q_heads * dim and q_stride % 8 == 0 and out_stride >= q_heads * dim and out_stride % 8 == 0
              and block_table.dtype is _int and block_table.is_contiguous() and block_table.get_device() == device and batch > 0
              and seq_lens.shape == (batch,) and seq_lens.dtype is _int and seq_lens.is_contiguous() and seq_lens.get_device() == device
              and q_starts.shape == (batch + 1,) and q_starts.dtype is _int and q_starts.is_contiguous() and q_starts.get_device() == device)
    except (AttributeError, TypeError, ValueError, IndexError):
        ok = False
    if ok:
        _call(_lib().syfi_paged_attention_block, device,
              _pack_attention(q.data_ptr(), q_stride, kv_cache.data_ptr(), pages, page_stride, block_table.data_ptr(), max_pages,
                              seq_lens.data_ptr(), q_starts.data_ptr(), batch, tokens, q_heads, heads, dim,
                              1.0 / math.sqrt(dim) if scale is None else float(scale), _window_of(window), out.data_ptr(), out_stride, _stream_of(stream, device)))
        return out
    pages, page_stride, kinds, heads, dim = _cache_of(kv_cache)
    dev = kv_cache.device
    if kinds != 2:
        raise ValueError("kv_cache must hold keys and values")
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be a 3-D tensor [tokens, q_heads, head_dim]")
    tokens, q_heads = q.shape[0], q.shape[1]
    if q_heads == 0 or q_heads % heads:
        raise ValueError(f"q has {q_heads} heads, expected a multiple of the cache's {heads}")
    q_stride = _tokens_of(q, "q", tokens, q_heads, dim, dev)
    out_stride = _tokens_of(out, "out", tokens, q_heads, dim, dev)
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("block_table must be a 2-D tensor [batch, max_pages]")
    batch, max_pages = block_table.shape
    table_ptr = _expect(block_table, "block_table", _int, (batch, max_pages), dev)
    lens_ptr = _expect(seq_lens, "seq_lens", _int, (batch,), dev)
    starts_ptr = _expect(q_starts, "q_starts", _int, (batch + 1,), dev)
    window = _window_of(window)
    if tokens and batch:
        _call(_lib().syfi_paged_attention_block, dev.index,
              _pack_attention(q.data_ptr(), q_stride, kv_cache.data_ptr(), pages, page_stride, table_ptr, max_pages, lens_ptr, starts_ptr, batch,
                              tokens, q_heads, heads, dim, 1.0 / math.sqrt(dim) if scale is None else float(scale), window, out.data_ptr(),
                              out_stride, _stream_ptr(stream, dev.index)))
    return out


def kv_check(device=None, stream=None):
    """Synchronise and raise :class:`MoeError` if an attention kernel gave up on a bounded wait."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(dev):
        _check(_lib().syfi_kv_check(_stream_ptr(stream, dev.index)))


__all__ = ["kv_cache_shape", "kv_check", "run_kv_read", "run_kv_write", "run_paged_attention"]
