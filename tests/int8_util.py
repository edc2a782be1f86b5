"""Inputs and bounds that the tests of the 8-bit operators share."""
import numpy as np

from oracle import int8_oracle as IO
from oracle import paged_oracle as PO
from paged_util import EPS, block_table, host, torch_type, words


def cache_of(rng, pages, page, block, kv_heads, d, spread=0.3):
    """Codes that reach 127 or so in every block, and scales that differ, in numpy."""
    codes = np.clip(np.rint(rng.standard_normal((pages, page, kv_heads, d)) * 35), -127, 127).astype(np.int8)
    return codes, (np.exp(spread * rng.standard_normal((pages, page // block, kv_heads))) / 35).astype(np.float32)


def attention_inputs(rng, dtype, heads, kv_heads, d, page, block, cached, fresh, spare=3, rows=None, gain=1.0, spread=0.3):
    """q on the device, codes and scales of keys and values, table, starts, lengths in numpy."""
    import torch
    total = np.asarray(cached) + np.asarray(fresh)
    pages = int(sum(-(-n // page) for n in total)) + spare
    starts = np.concatenate([[0], np.cumsum(fresh)])
    q = torch.from_numpy(rng.standard_normal((rows or max(1, int(starts[-1])), heads, d)).astype(np.float32) * gain).cuda().to(torch_type(dtype))
    k, ks = cache_of(rng, pages, page, block, kv_heads, d, spread)
    v, vs = cache_of(rng, pages, page, block, kv_heads, d, spread)
    return q, k, v, ks, vs, block_table(rng, total, page, pages), starts, total


def attention_bound(dtype, want, size, reach, d, floor=0.0):
    """How far an output may be from the exact one.

    The result's rounding: half a step, 2^-25 where f16 is subnormal.  A weight is 2^(s - m) over their sum.  Its exponent: s is d products in f32 whose sizes sum to at most `reach`, each
    addition off by 2^-24 of a partial sum (twice that where tensor cores truncate), then two products by scales: off by (d + 8) 2^-23 reach in all, which the weight
    carries relatively, numerator and sum alike; the exponential adds 2^-21.  A weight times its scale is rounded to f16 before it meets its code: half a step,
    2^-11.  The f32 sums of weights times codes add (1 + 64 joins) 2^-22 of `size`.

    `floor`, a row's keys times the cache's largest value: an f16 ends at 2^-24, so each weight is off by 2^-25 at least.  A row's largest is 2^7 times 1 or more
    (many tokens: 2^8), the block's scale over its power of two, which is at most 8 times the largest scale: 2^-25 * 2^-7 * 8 = 2^-29 of the largest value per key.  It shows
    where the one key that counts has a code of 0, and the next one a weight of 2^-49.
    """
    weight = 2 * (d + 8) * 2.0 ** -23 * reach + 2.0 ** -20 + 64 * 2.0 ** -22 + 2.0 ** -11
    return EPS[dtype] / 2 * np.abs(want) + np.minimum(weight, 1.0)[..., None] * size + (2.0 ** -25 if dtype == "f16" else 1e-30) + 2.0 ** -29 * floor


def wider(table, page, reach):
    """A table that goes on to `reach` tokens, which no sequence has: what the tables allow has a say in which kernels run."""
    return np.concatenate([table, np.full((len(table), max(0, reach // page - table.shape[1])), -1, table.dtype)], 1)


def check_attention(dtype, q, k, v, ks, vs, table, starts, lengths, scale=None, window=0, out=None, most=None, spread=None):
    """The operator on these inputs against the restatement; rows that belong to nobody against what was there before."""
    import torch
    from meganeura_b200 import ops
    scale = q.shape[2] ** -0.5 if scale is None else scale
    if out is None:
        out = torch.full(q.shape, 3.0, dtype=q.dtype, device="cuda")
    before = host(out).copy()
    d = [torch.from_numpy(x).cuda() for x in (k, v, ks, vs)]
    most = most or max(1, int(np.diff(starts).max()))
    page = k.shape[1]
    want, size, reach = PO.attention(host(q), IO.values(k, ks), IO.values(v, vs), table, starts, lengths, scale, window)
    nobody = np.isnan(want).all((1, 2)) & (np.arange(len(want)) >= min(int(starts[-1]), len(want)))
    want = want[~nobody]
    fine = ~np.isnan(want)
    bound = attention_bound(dtype, want, size[~nobody], reach[~nobody], q.shape[2], int(max(lengths)) * 127.0 * vs[np.isfinite(vs)].max())[fine]
    tables = [table]
    if max(lengths) <= table.shape[1] * page and most * (q.shape[1] // k.shape[2]) > 32:      # more than one kernel may take them, and together
        tables = [wider(table, page, 2 ** 20), wider(table, page, 2 ** 15 // len(table)), table]
    for t in tables:
        ops.paged_attention_int8(q, *d, words(t), words(starts), words(lengths), most, scale=scale, window=window, out=out)
        got = host(out)
        assert np.array_equal(got[nobody], before[nobody])
        got = got[~nobody]
        assert np.array_equal(np.isnan(got), np.isnan(want)), f"{np.isnan(got).sum()} NaN, {np.isnan(want).sum()} wanted"
        off = np.abs(got - want)[fine]
        assert np.isfinite(got[fine]).all()
        worst = (off - bound).max() if off.size else 0
        assert worst <= 0, f"off by {off.max():.3g}, {(off / bound).max():.2f} times the bound"
    return got
