"""Serving with 8-bit integers: torch-level entry points over the C ABI (mgq_quantize_rows, mgq_matmul_int8, mgq_paged_append_int8,
mgq_paged_attention_int8), reached as functions of `ops`.

A value is code * scale: int8 codes from -127 to 127, float32 scales, one for a row of a matrix or for a block of tokens and a head of a paged
cache.  As in paged.py every computation happens in libmgq, and a call asks once whether everything is as it should be.
"""
from __future__ import annotations

import functools

import torch

from ._lib import FMT_BF16, FMT_F16, FMT_F32, check, lib
from .paged import _is, _on, _pitch, _refuse, _table

_FORMATS = {torch.float32: FMT_F32, torch.float16: FMT_F16, torch.bfloat16: FMT_BF16}
_HALF = {torch.float16: FMT_F16, torch.bfloat16: FMT_BF16}
_i8, _i32, _f32 = torch.int8, torch.int32, torch.float32


@functools.lru_cache(maxsize=4096)
def _attention_workspace(heads: int, kv_heads: int, head_dim: int, max_fresh: int) -> int:
    return max(int(lib.mgq_paged_attention_int8_workspace(heads, kv_heads, head_dim, max_fresh)), 16)


def quantize_rows(x, out=None, stream=None):
    """Rows of x [rows, k] (float32, float16, bfloat16; rows any distance apart) as codes [rows, k] int8 and scales [rows] float32 (mgq_quantize_rows).

    Activations get a scale per token, weights [n, k] one per channel.  out: (codes, scales) to write to.
    """
    device, dtype = x.get_device(), x.dtype
    if device < 0 or x.dim() != 2 or dtype not in _FORMATS:
        raise ValueError("x must be a [rows, k] CUDA tensor of float32, float16 or bfloat16; the library has no CPU path")
    rows, k = x.shape
    pitch = _pitch("x", x, device, k)
    if out is not None and not (_is(out[0], _i8, device, (rows, k)) and _is(out[1], _f32, device, (rows,))):
        _refuse(device, codes=(out[0], _i8, (rows, k)), scales=(out[1], _f32, (rows,)))

    def call(sp):
        codes, scales = (x.new_empty((rows, k), dtype=_i8), x.new_empty(rows, dtype=_f32)) if out is None else out
        check(lib.mgq_quantize_rows(x.data_ptr(), _FORMATS[dtype], pitch, codes.data_ptr(), scales.data_ptr(), rows, k, sp))
        return codes, scales
    return _on(device, stream, call)


def _result_pitch(name: str, t, dtype, device: int, m: int, n: int) -> int:
    if t.dtype is not dtype or t.shape != (m, n):
        raise ValueError(f"{name} must be a {dtype} tensor of shape {(m, n)}, not {tuple(t.shape)} {t.dtype}")
    return _pitch(name, t, device, n)


def matmul_int8(a, a_scales, w, w_scales, addend=None, out=None, dtype=None, stream=None):
    """(a @ w.T) * a_scales[:, None] * w_scales (+ addend), the product in whole numbers (mgq_matmul_int8).

    a: [m, k] int8 codes of activations, a_scales: [m] float32; w: [n, k] int8, w_scales: [n] float32, as quantize_rows writes them.  k: a multiple
    of 16.  The result [m, n] has the type of out or addend or `dtype` (bfloat16 where none is given); out and addend have one type and rows any distance apart; out may be
    addend.
    """
    device = a.get_device()
    if device < 0 or a.dim() != 2 or w.dim() != 2:
        raise ValueError("a and w must be [m, k] and [n, k] CUDA tensors; the library has no CPU path")
    (m, k), n = a.shape, w.shape[0]
    if not (_is(a, _i8, device, (m, k)) and _is(w, _i8, device, (n, k)) and _is(a_scales, _f32, device, (m,)) and _is(w_scales, _f32, device, (n,))):
        _refuse(device, a=(a, _i8, (m, k)), w=(w, _i8, (n, k)), a_scales=(a_scales, _f32, (m,)), w_scales=(w_scales, _f32, (n,)))
    if dtype is None:
        dtype = out.dtype if out is not None else addend.dtype if addend is not None else torch.bfloat16
    form = _FORMATS.get(dtype)
    if form is None:
        raise ValueError(f"the result must be float32, float16 or bfloat16, not {dtype}")
    out_pitch = n if out is None else _result_pitch("out", out, dtype, device, m, n)
    add_pitch = 0 if addend is None else _result_pitch("addend", addend, dtype, device, m, n)

    def call(sp):
        o = a.new_empty((m, n), dtype=dtype) if out is None else out
        check(lib.mgq_matmul_int8(a.data_ptr(), a_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), None if addend is None else addend.data_ptr(), o.data_ptr(),
                                  form, m, k, n, add_pitch, out_pitch, sp))
        return o
    return _on(device, stream, call)


def _caches(k_cache, v_cache, k_scales, v_scales):
    device, shape = k_cache.get_device(), k_cache.shape
    if device < 0:
        raise ValueError("a paged cache lives on the GPU; the library has no CPU path")
    if len(shape) != 4 or k_cache.dtype is not _i8 or not (k_cache.is_contiguous() and _is(v_cache, _i8, device, shape)):
        raise ValueError("k_cache and v_cache must be alike: contiguous int8 [pages, page_size, kv_heads, head_dim] on one device")
    pages, page_size, kv_heads, d = shape
    blocks = k_scales.shape[1] if k_scales.dim() == 3 else 0
    scales = (pages, blocks, kv_heads)
    if blocks < 1 or page_size % blocks or not (_is(k_scales, _f32, device, scales) and _is(v_scales, _f32, device, scales)):
        raise ValueError(f"k_scales and v_scales must be alike: contiguous float32 [{pages}, page_size / block, {kv_heads}] on cuda:{device}")
    return device, pages, page_size, kv_heads, d, page_size // blocks


def paged_append_int8(q, k, v, positions, slots, k_cache, v_cache, k_scales, v_scales, theta: float = 0.0, q_out=None, q_dtype=None, stream=None):
    """Rows of keys (rotated where theta > 0) and values into a cache of 8-bit codes, and the rotated queries (mgq_paged_append_int8).

    As paged_append, but for the caches: int8 codes [pages, page_size, kv_heads, head_dim] and float32 scales [pages, page_size / block, kv_heads], updated
    together.  Rows may stand in any order; fastest is a PagedStep's, where those of one block of tokens stand one behind another.  q, k, v: float32, float16 or bfloat16; returns
    q_out [rows, heads, head_dim], float16 or bfloat16 (q_dtype; the sources' type or bfloat16 where neither is given).
    """
    device, pages, page_size, kv_heads, d, block = _caches(k_cache, v_cache, k_scales, v_scales)
    rows, src = k.shape[0], k.dtype
    dst = q_out.dtype if q_out is not None else q_dtype or (src if src in _HALF else torch.bfloat16)
    if dst not in _HALF or src is not _f32 and src is not dst or v.dtype is not src or q is not None and q.dtype is not src:
        raise ValueError("q, k and v must have one type: float32 or that of the rotated queries, float16 or bfloat16")
    if k.shape != (rows, kv_heads, d) or v.shape != k.shape or q is not None and (q.dim() != 3 or q.shape[0] != rows or q.shape[2] != d):
        raise ValueError(f"k and v must be [rows, {kv_heads}, {d}] and q [rows, heads, {d}], not {tuple(k.shape)}, {tuple(v.shape)}, {None if q is None else tuple(q.shape)}")
    if not (_is(positions, _i32, device, (rows,)) and _is(slots, _i32, device, (rows,))):
        _refuse(device, positions=(positions, _i32, (rows,)), slots=(slots, _i32, (rows,)))
    heads = 0 if q is None else q.shape[1]
    q_pitch, k_pitch, v_pitch = 0 if q is None else _pitch("q", q, device, heads * d), _pitch("k", k, device, kv_heads * d), _pitch("v", v, device, kv_heads * d)
    if q is not None and q_out is not None and not _is(q_out, dst, device, (rows, heads, d)):
        _refuse(device, q_out=(q_out, dst, (rows, heads, d)))

    def call(sp):
        out = None if q is None else k_cache.new_empty((rows, heads, d), dtype=dst) if q_out is None else q_out
        check(lib.mgq_paged_append_int8(None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), _FORMATS[src], positions.data_ptr(), slots.data_ptr(),
                                        None if out is None else out.data_ptr(), _HALF[dst], k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                        rows, heads, kv_heads, d, q_pitch, k_pitch, v_pitch, page_size, pages, block, theta, sp))
        return out
    return _on(device, stream, call)


def paged_attention_int8(q, k_cache, v_cache, k_scales, v_scales, table, starts, lengths, max_fresh: int, scale: float | None = None, window: int = 0, out=None, stream=None):
    """Attention of a step's new tokens over their sequences' pages of 8-bit codes (mgq_paged_attention_int8).

    As paged_attention, but for the caches (see paged_append_int8); q [rows, heads, head_dim] and out are float16 or bfloat16.
    """
    device, pages, page_size, kv_heads, d, block = _caches(k_cache, v_cache, k_scales, v_scales)
    dtype = q.dtype
    if dtype not in _HALF or q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"q must be [rows, heads, {d}] float16 or bfloat16, not {tuple(q.shape)} {dtype}")
    rows, heads, _ = q.shape
    _, sequences, width = _table(table)
    if table.get_device() != device or not (_is(starts, _i32, device, (sequences + 1,)) and _is(lengths, _i32, device, (sequences,))):
        _refuse(device, table=(table, _i32, (None, None)), starts=(starts, _i32, (sequences + 1,)), lengths=(lengths, _i32, (sequences,)))
    if window < 0 or max_fresh < 1:
        raise ValueError(f"window {window} is negative or max_fresh {max_fresh} not positive")
    if window >> 31:                                    # no sequence is that long
        window = 0
    most = min(max_fresh, 0xFFFFFFFF)
    q_pitch = _pitch("q", q, device, heads * d)
    if out is not None and (out.dtype is not dtype or out.shape != q.shape):
        raise ValueError("out must have the shape and the type of q")

    def call(sp):
        o = q.new_zeros((rows, heads, d)) if out is None else out
        room = q.new_empty(_attention_workspace(heads, kv_heads, d, most), dtype=torch.uint8)
        check(lib.mgq_paged_attention_int8(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), _HALF[dtype], table.data_ptr(),
                                           starts.data_ptr(), lengths.data_ptr(), o.data_ptr(), sequences, rows, most, heads, kv_heads, d, page_size, pages, block, width,
                                           q_pitch, _pitch("out", o, device, heads * d), d ** -0.5 if scale is None else scale, window, room.data_ptr(), sp))
        return o
    return _on(device, stream, call)
