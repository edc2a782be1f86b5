"""Inputs and bounds that the tests of the paged operators share."""
import numpy as np

from oracle import paged_oracle as PO

EPS = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def host(t):
    """A tensor's values in numpy, 16-bit ones as f32."""
    import torch
    return t.float().cpu().numpy() if t.dtype in (torch.float16, torch.bfloat16) else t.cpu().numpy()


def words(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int64).astype(np.int32))).cuda()


def block_table(rng, tokens, page, pages, width=None):
    """[sequences, width] with the pages of tokens[s] tokens each, shuffled; the rest names no page."""
    need = [-(-int(n) // page) for n in tokens]
    order = rng.permutation(pages)
    table, at = np.full((len(tokens), width or max(1, max(need))), -1, np.int64), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table


def attention_inputs(rng, dtype, heads, kv_heads, d, page, cached, fresh, spare=3, rows=None, gain=1.0):
    """q, k_cache, v_cache on the device, table, starts, lengths in numpy."""
    import torch
    t = torch_type(dtype)
    total = np.asarray(cached) + np.asarray(fresh)
    pages = int(sum(-(-n // page) for n in total)) + spare
    starts = np.concatenate([[0], np.cumsum(fresh)])
    q = torch.from_numpy(rng.standard_normal((rows or int(starts[-1]), heads, d)).astype(np.float32) * gain).cuda().to(t)
    k, v = (torch.from_numpy(rng.standard_normal((pages, page, kv_heads, d)).astype(np.float32)).cuda().to(t) for _ in range(2))
    return q, k, v, block_table(rng, total, page, pages), starts, total


def attention_bound(dtype, want, size, reach, d):
    """How far an output may be from the exact one.

    One rounding of the result: half a step.  A weight is 2^(s - m) over their sum: s has d products in f32 whose sizes sum to at most
    `reach` (scaled), each addition off by 2^-24 of a partial sum (twice that where tensor cores truncate), so an exponent is off by (d + 8) 2^-23 reach,
    which a weight carries relatively, numerator and sum alike; the exponential adds 2^-21.  16-bit kernels round a weight to the type before
    it meets its value: half a step of the type.  The f32 sums of weights * values add (1 + 64 joins) 2^-22 of `size`.
    """
    half = EPS[dtype] / 2
    weight = 2 * (d + 8) * 2.0 ** -23 * reach + 2.0 ** -20 + 64 * 2.0 ** -22 + (half if dtype != "f32" else 0.0)
    return half * np.abs(want) + np.minimum(weight, 1.0)[..., None] * size + 2.0 ** -24 * size + 1e-30


def check_attention(dtype, q, k, v, table, starts, lengths, got, scale, window=0, before=None):
    """`got` against the oracle; rows that belong to nobody against what was there before."""
    want, size, reach = PO.attention(host(q), host(k), host(v), table, starts, lengths, scale, window)
    nobody = np.isnan(want).all((1, 2))
    got = host(got)
    if before is not None:
        assert np.array_equal(got[nobody], before[nobody])
    off, bound = np.abs(got[~nobody] - want[~nobody]), attention_bound(dtype, want, size, reach, q.shape[2])[~nobody]
    assert np.isfinite(got[~nobody]).all()
    worst = (off - bound).max() if off.size else 0
    assert worst <= 0, f"off by {off.max():.3g}, {(off / bound).max():.2f} times the bound"
