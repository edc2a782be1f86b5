"""The operators over a paged cache and from logits to tokens, at values and lengths where their kernels' arithmetic or order could go wrong."""
import math

import numpy as np
import pytest

from oracle import paged_oracle as PO
from paged_util import host

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- probabilities

def check_probs(logits, temperature):
    import torch
    from meganeura_b200 import ops
    t = np.asarray(temperature, np.float32)
    got = host(ops.token_probs(torch.from_numpy(logits).cuda(), torch.from_numpy(t).cuda()))
    want = PO.probs(logits, t)
    assert np.isfinite(got).all()
    # the exponent (x - m) / t is off by 2^-22 of its size, which is at most 104 where a weight is not below f32's range; the exponential 2^-22, the
    # sum 2^-18.  Below f32's normal range a weight is a multiple of 2^-149: expf's two units there, and half a unit of the product with 1 / sum
    clean = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    top = clean.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        spread = np.nan_to_num(np.minimum(104.0, (top - clean) / np.maximum(t, 1e-30)[:, None]), nan=0.0)
    off, bound = np.abs(got - want), want * (2.0 ** -22 * (spread + 1) + 2.0 ** -18) + 2.5 * 2.0 ** -149
    at = np.unravel_index((off - bound).argmax(), off.shape)
    assert off[at] <= bound[at], (at, got[at], want[at])


@pytest.mark.parametrize("rows,vocab", [(2, 151936), (3, 70001), (80, 40000), (2, 300004), (4, 32768), (3, 5001)])
@pytest.mark.parametrize("kept", ["late", "top", "prefix", "alternating"])
def test_token_probs_of_masked_rows(rows, vocab, kept):
    """-inf (or NaN) in all but a few columns, as masks of a grammar, top-k or padding of the vocabulary leave them, with small and large temperatures."""
    rng = np.random.default_rng(vocab)
    logits = np.full((rows, vocab), -np.inf, np.float32)
    if kept != "prefix":
        logits[1::2] = np.nan
    for r in range(rows):
        n = min(300, vocab // 4)
        cols = {"late": np.arange(vocab - n, vocab), "top": rng.choice(vocab, 50, replace=False), "prefix": np.arange(n), "alternating": np.arange(r % 2, vocab, 2)}[kept]
        logits[r, cols] = rng.standard_normal(len(cols)) * 3 - [1, 10, 26, 100, 200, 300][r % 6]
    for t in (0.05, 0.3, 1.0, 4.0):
        check_probs(logits, [t] * rows)
    check_probs(logits, rng.choice([0.0, 0.1, 2.0], rows))


@pytest.mark.parametrize("vocab", [151936, 70001])
def test_token_probs_of_long_rows_with_infinities_and_ties(vocab):
    rng = np.random.default_rng(vocab)
    logits = (rng.standard_normal((9, vocab)) * 3 - 50).astype(np.float32)
    logits[0] = -np.inf                                            # nothing is left
    logits[1] = np.nan
    logits[2, [vocab - 1, vocab // 2, 70]] = np.inf                # these share the row
    logits[3, :vocab // 3], logits[3, vocab - 5] = -np.inf, np.inf
    logits[4, [vocab - 2, vocab // 2 + 1, vocab // 4]] = 9.0       # the largest, in several CTAs' shares
    logits[5, :] = -3e38                                           # the type's lowest values as a mask
    logits[5, vocab // 2:vocab // 2 + 40] = -70.0
    logits[6, :] = np.finfo(np.float32).min
    logits[7, ::2] = np.nan
    logits[8, :vocab - 1] = -np.inf
    for t in (1.0, 0.1, 0.0):
        check_probs(logits, [t] * 9)


@pytest.mark.parametrize("rows,vocab", [(2, 151936), (3, 70001), (4, 32768), (3, 5001), (2, 7), (80, 40000)])
def test_token_probs_at_an_infinite_temperature_and_of_values_at_the_range_s_ends(rows, vocab):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(vocab)
    big = np.finfo(np.float32).max
    for masked in (False, True):
        logits = (rng.standard_normal((rows, vocab)) * 20).astype(np.float32)
        logits[1, ::2] = -big                                      # a finite mask is a number like any other
        logits[0, -1] = big
        if masked:
            logits[:, 1::3] = -np.inf
            logits[1, 4::7] = np.nan
        seen = np.where(np.isnan(logits), -np.inf, logits) > -np.inf
        got = host(ops.token_probs(torch.from_numpy(logits).cuda(), torch.full((rows,), math.inf, device="cuda")))
        want = seen / seen.sum(1, keepdims=True)
        # a difference of at most 2^129 times 2^-149 is an exponent of 2^-20 at most, in the weight and in the sum; the sum adds 2^-18
        assert (np.abs(got - want) <= want * (2.0 ** -19 + 2.0 ** -18)).all()
        # the largest differences there are: 2 * 3.4e38 / 1e38 = 6.8
        t = np.full(rows, 1e38, np.float32)
        got = host(ops.token_probs(torch.from_numpy(logits).cuda(), torch.from_numpy(t).cuda()))
        want = PO.probs(logits, t)
        assert (np.abs(got - want) <= want * (2.0 ** -22 * 8 + 2.0 ** -18)).all()


# ---------------------------------------------------------------------------------------------- attention: units in every order

def attend(q, k, v, table, starts, lengths, most, **kw):
    from meganeura_b200 import ops
    from paged_util import words
    out = ops.paged_attention(q, k, v, words(table), words(starts), words(lengths), most, **kw)
    ops.device_status()                                            # no wait inside the kernels ran out
    return out


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64)])
def test_attention_of_many_tokens_whose_units_often_have_no_keys(dtype, d):
    """Sequences without tokens in the cache (lengths of 0, pages that nobody has) between others, one behind another and at both ends."""
    import torch
    rng = np.random.default_rng(d)
    fresh = np.tile([40, 90, 33, 200, 64], 120)
    empty = np.array([(s // 5) % 3 != 1 or s % 5 == 2 for s in range(len(fresh))])
    from paged_util import attention_inputs, check_attention
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, 4, 2, d, 16, np.where(empty, 0, rng.integers(0, 300, len(fresh))), fresh)
    lengths = np.where(empty, 0, lengths)
    first = attend(q, k, v, table, starts, lengths, 200)
    for s in np.flatnonzero(empty):
        assert (first[int(starts[s]):int(starts[s + 1])] == 0).all()
    for s in np.flatnonzero(~empty)[::9]:
        rows = slice(int(starts[s]), int(starts[s + 1]))
        check_attention(dtype, q[rows], k, v, table[s:s + 1], [0, fresh[s]], [lengths[s]], first[rows], d ** -0.5)
    for _ in range(5):
        assert torch.equal(attend(q, k, v, table, starts, lengths, 200), first)


@pytest.mark.parametrize("dtype,heads,kv_heads,d", [("bf16", 8, 2, 128), ("f16", 3, 1, 64), ("bf16", 2, 2, 80)])
def test_attention_of_very_many_short_units_of_many_tokens(dtype, heads, kv_heads, d):
    """Units of one or two blocks of keys, some with one tile and some with two: every wait of the kernel's roles meets its next phase at once."""
    import torch
    from paged_util import attention_inputs, check_attention
    rng = np.random.default_rng(heads)
    fresh = rng.integers(33 * kv_heads // heads + 1, 70, 1500)
    cached = rng.choice([0, 1, 60, 127, 128, 200], 1500)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 8, cached, fresh)
    first = attend(q, k, v, table, starts, lengths, 70)
    for s in range(0, 1500, 97):
        rows = slice(int(starts[s]), int(starts[s + 1]))
        check_attention(dtype, q[rows], k, v, table[s:s + 1], [0, fresh[s]], [lengths[s]], first[rows], d ** -0.5)
    for _ in range(10):
        assert torch.equal(attend(q, k, v, table, starts, lengths, 70), first)


@pytest.mark.parametrize("dtype,heads,kv_heads,d,window", [("bf16", 8, 2, 128, 0), ("f16", 4, 4, 64, 0), ("f16", 8, 1, 64, 500)])
def test_attention_of_units_whose_second_tile_has_nothing_to_do(dtype, heads, kv_heads, d, window):
    """Up to 128 pairs over long sequences: the idle tile hands on the stages of every block, for many units one behind another and beside full ones."""
    import torch
    from paged_util import attention_inputs, check_attention
    rng = np.random.default_rng(heads + d)
    g = heads // kv_heads
    fresh = np.array([128 // g, 33 // g + 1, 200, 100 // g, 128 // g + 1, 64 // g] * 10)
    cached = rng.integers(1500, 4000, len(fresh))
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, cached, fresh)
    first = attend(q, k, v, table, starts, lengths, 200, window=window)
    for s in range(0, len(fresh), 7):
        i = int(rng.integers(0, fresh[s]))
        r = int(starts[s]) + i                                     # the row alone, as the last token of its sequence
        check_attention(dtype, q[r:r + 1], k, v, table[s:s + 1], [0, 1], [cached[s] + i + 1], first[r:r + 1], d ** -0.5, window)
    for _ in range(10):
        assert torch.equal(attend(q, k, v, table, starts, lengths, 200, window=window), first)


# ---------------------------------------------------------------------------------------------- attention: scores and weights at the range's ends

@pytest.mark.parametrize("dtype,heads,kv_heads,d,fresh", [
    ("bf16", 8, 2, 128, 60), ("f16", 8, 2, 128, 60), ("f16", 3, 1, 64, 200), ("bf16", 4, 4, 80, 300), ("bf16", 8, 2, 128, 1), ("f16", 8, 2, 64, 5), ("f16", 4, 2, 256, 3),
    ("f32", 4, 1, 128, 1), ("f32", 4, 2, 64, 5), ("f32", 8, 2, 128, 60), ("f32", 2, 1, 256, 7), ("bf16", 3, 1, 20, 9),
])
@pytest.mark.parametrize("scale", [0.0883883, 1.0, 37.0])
def test_attention_with_scores_far_beyond_what_a_weight_distinguishes(dtype, heads, kv_heads, d, fresh, scale):
    """Scores of 2^20 to 2^50, whole steps of 2^17 and more apart: a row is the mean of the values whose score is the largest that it sees."""
    import torch
    from paged_util import EPS, attention_inputs, words
    rng = np.random.default_rng(d + fresh)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 16, [500, 90], [fresh, fresh])
    a, b = (2.0 ** 13, 2.0 ** 8) if dtype == "f16" else (2.0 ** 22, 2.0 ** 20)
    level = rng.integers(1, 100, k.shape[:3])
    level[rng.random(level.shape) < 0.02] = 100                   # the same score more than once
    q.zero_(), k.zero_()
    q[..., 3] = a
    for sign in (1.0, -1.0):                                       # the largest far above 0, and far below
        k[..., 3] = torch.from_numpy(sign * b * level).to(k)
        got = host(attend(q, k, v, table, starts, lengths, fresh, scale=scale))
        values = host(v).astype(np.float64)
        for s in range(2):
            slots = table[s, np.arange(lengths[s]) // 16] * 16 + np.arange(lengths[s]) % 16
            lv, vv = sign * level.reshape(-1, kv_heads)[slots], values.reshape(-1, kv_heads, d)[slots]
            for i in {0, 1, fresh // 2, fresh - 1} & set(range(fresh)):
                n = lengths[s] - fresh + i + 1
                for h in range(heads):
                    o = h * kv_heads // heads
                    best = lv[:n, o] == lv[:n, o].max()
                    want, size = vv[:n, o][best].mean(0), np.abs(vv[:n, o][best]).mean(0)
                    # equal weights: half a step of the result, and f32 sums of at most 100 values.  Relative to a maximum that is itself rounded a weight of many
                    # tokens is 2^(score - maximum) with an exponent other than 0, and then rounded to its type, while the sum has it unrounded: half a step more
                    rounded = EPS[dtype] / 2 if dtype != "f32" and fresh * heads // kv_heads > 32 else 0.0
                    assert (np.abs(got[int(starts[s]) + i, h] - want) <= EPS[dtype] / 2 * np.abs(want) + (rounded + 2.0 ** -17) * size + 2.0 ** -24).all(), (sign, s, i, h)


@pytest.mark.parametrize("dtype,heads,kv_heads,d,fresh", [("bf16", 8, 2, 128, 60), ("f16", 3, 1, 64, 200), ("f16", 8, 2, 128, 1), ("f32", 4, 2, 64, 40), ("f32", 4, 2, 64, 1)])
def test_attention_whose_first_keys_score_far_below_the_others(dtype, heads, kv_heads, d, fresh):
    """Scores of about -2^30 for the first 300 keys: while only they have been seen the maximum is that low, and nothing of it may stay."""
    from paged_util import EPS, attention_inputs
    rng = np.random.default_rng(fresh)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 16, [900], [fresh])
    a, b = (2.0 ** 13, 2.0 ** 14) if dtype == "f16" else (2.0 ** 16, 2.0 ** 16)
    q[..., 3], k[..., 3] = a, 0.0
    slots = table[0, np.arange(lengths[0]) // 16] * 16 + np.arange(lengths[0]) % 16
    import torch
    k.flatten(0, 1)[torch.from_numpy(slots[:300]).cuda(), :, 3] = -b
    want, size, _ = PO.attention(host(q), host(k), host(v), table, starts, lengths, d ** -0.5)
    got = host(attend(q, k, v, table, starts, lengths, fresh))
    # half a step of the result and of a weight; scores of the others: 64 to 128 products, a few units each of 2^-24 * 60
    assert (np.abs(got - want) <= EPS[dtype] / 2 * (np.abs(want) + size) + 2.0 ** -13 * size + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("bf16", 80)])
def test_attention_of_many_tokens_whose_rows_are_all_computed_again(dtype, d):
    """An infinite value that every row sees, in one column: the others are as without it.  One that only the last token sees: nobody else changes."""
    import torch
    from paged_util import attention_inputs, check_attention
    rng = np.random.default_rng(d)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, 8, 2, d, 32, [6000, 40], [130, 70])
    clean = attend(q, k, v, table, starts, lengths, 130)
    flat, at = v.flatten(0, 1), int(table[0, 0]) * 32 + 5
    old = flat[at, 1, 7].clone()
    flat[at, 1, 7] = math.inf
    got = attend(q, k, v, table, starts, lengths, 130)
    assert not torch.isfinite(got[:130, 4:, 7]).any()
    got[:130, 4:, 7] = clean[:130, 4:, 7]
    flat[at, 1, 7] = old
    for i in (0, 64, 129):
        check_attention(dtype, q[i:i + 1], k, v, table[:1], [0, 1], [6001 + i], got[i:i + 1], d ** -0.5)
    assert torch.equal(got[130:], clean[130:])
    at = int(table[0, 6129 // 32]) * 32 + 6129 % 32
    flat[at, 0, 3] = math.nan
    got = attend(q, k, v, table, starts, lengths, 130)
    assert torch.isnan(got[129, :4, 3]).all()
    for i in (0, 65, 128):
        check_attention(dtype, q[i:i + 1], k, v, table[:1], [0, 1], [6001 + i], got[i:i + 1], d ** -0.5)


def test_attention_waits_for_rows_that_are_computed_again_however_many():
    """A value that every row sees is infinite: all rows of every unit, one after another over 12000 keys, while the kernel's other roles wait."""
    import torch
    from paged_util import attention_inputs, check_attention
    rng = np.random.default_rng(31)
    q, k, v, table, starts, lengths = attention_inputs(rng, "bf16", 32, 8, 128, 64, [12000], [1200])
    clean = attend(q, k, v, table, starts, lengths, 1200)
    at = int(table[0, 1]) * 64 + 9
    old = v.flatten(0, 1)[at, :, 77].clone()
    v.flatten(0, 1)[at, :, 77] = -math.inf
    got = attend(q, k, v, table, starts, lengths, 1200)            # asks for the waits that ran out
    v.flatten(0, 1)[at, :, 77] = old
    assert not torch.isfinite(got[..., 77]).any()
    got[..., 77] = clean[..., 77]
    for i in rng.integers(0, 1200, 12).tolist():
        check_attention("bf16", q[i:i + 1], k, v, table, [0, 1], [12001 + i], got[i:i + 1], 128 ** -0.5)


@pytest.mark.parametrize("dtype,heads,kv_heads,d,fresh", [("f16", 8, 2, 128, 1), ("f16", 8, 2, 64, 5), ("f16", 4, 2, 256, 1), ("f16", 8, 2, 128, 60), ("f16", 3, 1, 64, 200),
                                                          ("bf16", 8, 2, 128, 1), ("bf16", 8, 2, 128, 60), ("f32", 4, 2, 64, 1), ("f32", 4, 2, 64, 40)])
@pytest.mark.parametrize("score", [-10.0, -17.0, -20.0, -24.0])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_attention_keeps_small_weights_beside_one_that_dominates(dtype, heads, kv_heads, d, fresh, score, place):
    """20000 keys of weight e^score beside one of weight 1, whose value is 0: together they are all of the result."""
    from paged_util import EPS, attention_inputs
    rng = np.random.default_rng(d + fresh)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, [20000], [fresh])
    q.zero_(), k.zero_()
    q[..., 1], k[..., 1] = 1.0, score
    v.abs_().mul_(32.0).add_(64.0)
    at = {"first": 0, "middle": 9001, "last": 20000}[place]
    slot = table[0, at // 32] * 32 + at % 32
    k.flatten(0, 1)[slot], v.flatten(0, 1)[slot] = 0.0, 0.0
    got = host(attend(q, k, v, table, starts, lengths, fresh, scale=1.0))
    slots = table[0, np.arange(lengths[0]) // 32] * 32 + np.arange(lengths[0]) % 32
    values = host(v).astype(np.float64).reshape(-1, kv_heads, d)[slots]
    many = fresh * (heads // kv_heads) > 32
    for i in sorted({0, fresh // 3, fresh - 1}):
        n = lengths[0] - fresh + i + 1
        w = np.full(n, math.exp(score))
        w[at] = 1.0
        for h in range(0, heads, 2):
            x = values[:n, h * kv_heads // heads]
            want = w @ x / w.sum()
            # A weight is off by 2^-17 (the exponent's rounding and the exponential), of many tokens by half a step of its type; f16 rounds it to a multiple of 2^-32
            # (many tokens) or 2^-39 (few) of the largest.  A sum that holds the 1 first loses up to 2^-25 with each addition behind it: of up to 600 parts that
            # are joined one by one, and in a part of a few dozen more, in numerator and denominator.  The result is rounded once, in f16 to a multiple of 2^-24.
            least = 0.0 if dtype != "f16" else 2.0 ** -33 if many else 2.0 ** -40
            weight = 2.0 ** -17 + 2 * 640 * 2.0 ** -25 + (EPS[dtype] / 2 if many and dtype != "f32" else 0.0)
            bound = EPS[dtype] / 2 * want + weight * want + least * x.sum(0) / w.sum() + 2.0 ** -25
            off = np.abs(got[i, h] - want)
            assert (off <= bound).all(), (i, h, (off / bound).max())


# ---------------------------------------------------------------------------------------------- what the Python side hands on

def test_whole_numbers_beyond_32_bits_are_refused_or_mean_what_they_say():
    import torch
    from meganeura_b200 import ops
    from paged_util import attention_inputs, words
    rng = np.random.default_rng(3)
    w = words(np.zeros(2))
    for page_size, rows in ((2 ** 32 + 16, 8), (-16, 8), (16, 2 ** 32 + 8)):
        with pytest.raises(ValueError):
            ops.paged_plan(w, w, words(np.zeros((2, 4))), w.clone(), words(np.zeros(8)), w[:1].clone(), page_size, rows)
    with pytest.raises(ValueError):
        ops.paged_trim(w, words(np.zeros((2, 4))), w.clone(), words(np.zeros(8)), w[:1].clone(), 2 ** 32 + 16)
    q, k, v, table, starts, lengths = attention_inputs(rng, "bf16", 4, 2, 64, 16, [60, 9], [50, 1])
    want = attend(q, k, v, table, starts, lengths, 50)
    for window in (2 ** 31, 2 ** 32 + 5, 2 ** 63):
        assert torch.equal(attend(q, k, v, table, starts, lengths, 50, window=window), want)
    assert torch.equal(attend(q, k, v, table, starts, lengths, 2 ** 32 + 1), want)


def test_verified_tokens_of_rows_behind_the_last_sequence_are_none():
    import torch
    from meganeura_b200 import ops
    from paged_util import words
    p = torch.softmax(torch.randn(40, 100, device="cuda"), 1)
    for _ in range(3):
        torch.full((4000,), 77, dtype=torch.int32, device="cuda")                      # what new tensors may hold
        got = ops.verify_drafts(p, None, words(np.arange(40)), words([0, 3, 5]), torch.rand(40, device="cuda"), torch.rand(2, device="cuda"))
        assert got[0].shape == got[1].shape == (2,) and got[2].shape == (40,) and (got[2][5:] == ops.NO_TOKEN).all()
