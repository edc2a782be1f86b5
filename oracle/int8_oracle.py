"""Rows of 8-bit codes and paged caches of them, restated in numpy: one row, block and head at a time, in 64 bits but for the scales, whose f32 roundings are
part of the definition (a code is the rounding of a quotient by the scale that is stored)."""
import numpy as np

LEAST = np.float32(2.0 ** -100)


def scale_of(top):
    top = np.float32(top)
    return np.float32(0) if top < LEAST else np.float32(top * (np.float32(1) / np.float32(127)))


def inverse_of(scale):
    scale = np.float32(scale)
    return np.float32(1) / scale if scale > 0 and np.isfinite(scale) else np.float32(0)


def codes_of(x, scale):
    """Codes of f32 values by a scale, the product with its inverse rounded to f32 as the definition has it."""
    with np.errstate(invalid="ignore"):
        y = np.rint(np.asarray(x, np.float32) * inverse_of(scale))
    return np.where(np.isnan(y), 0, y).astype(np.int8)


def quantize_rows(x):
    x = np.asarray(x, np.float32)
    scales = np.array([scale_of(np.abs(r).max()) for r in x], np.float32)      # max keeps a NaN
    return np.stack([codes_of(r, s) for r, s in zip(x, scales)]), scales


def matmul(a, a_scales, w, w_scales, addend=None):
    y = (a.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64) * a_scales.astype(np.float64)[:, None] * w_scales.astype(np.float64)
    return y if addend is None else y + addend


def append(cache, scales, x, slots):
    """Rows x [rows, kv_heads, d] into copies of a cache's codes and scales."""
    pages, page, kv_heads, d = cache.shape
    block = page // scales.shape[1]
    cache, scales = cache.reshape(-1, block, kv_heads, d).copy(), scales.reshape(-1, kv_heads).copy()
    rows = {}
    for r, slot in enumerate(np.asarray(slots, np.int64)):
        if 0 <= slot < pages * page:
            rows.setdefault(slot // block, []).append((slot % block, r))
    for b, placed in rows.items():
        at, r = [p[0] for p in placed], [p[1] for p in placed]
        for h in range(kv_heads):
            old = np.float32(0) if 0 in at else scales[b, h]
            new = np.maximum(old, scale_of(np.abs(x[r, h].astype(np.float32)).max()))     # NaN stays
            if 0 not in at and not (old == new):
                ratio = np.float32(old / new) if inverse_of(new) else np.float32(0)
                held = [i for i in range(block) if i not in at]
                cache[b, held, h] = np.rint(cache[b, held, h].astype(np.float32) * ratio).astype(np.int8)
            cache[b, at, h] = codes_of(x[r, h], new)
            scales[b, h] = new
    return cache.reshape(pages, page, kv_heads, d), scales.reshape(pages, page // block, kv_heads)


def values(cache, scales):
    """A cache's values in 64 bits."""
    pages, page, kv_heads, d = cache.shape
    with np.errstate(invalid="ignore"):
        return (cache.reshape(pages, scales.shape[1], -1, kv_heads, d).astype(np.float64) * scales.astype(np.float64)[:, :, None, :, None]).reshape(cache.shape)
