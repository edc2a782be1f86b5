"""The 8-bit operators at the ends of what their documentation allows."""
import numpy as np
import pytest

from int8_util import attention_bound, attention_inputs, cache_of, check_attention, wider
from oracle import int8_oracle as IO
from oracle import paged_oracle as PO
from paged_util import EPS, block_table, host, words

pytestmark = pytest.mark.gpu


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (32, 2, 128), (9, 3, 80), (8, 1, 256)])
@pytest.mark.parametrize("fresh", [1, 3, 60])
def test_keys_that_are_infinite_make_their_rows_nan(dtype, heads, kv_heads, d, fresh):
    """Their block's scale is infinite and its codes are zeros, so that a score is 0 times infinity, never an infinity with a sign."""
    rng = np.random.default_rng(d + fresh)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, 16, [300] * 4, [fresh] * 4, gain=3.0)
    for s in range(4):
        k[table[s, 3], :16], ks[table[s, 3], 0] = 0, np.inf
    got = check_attention(dtype, q, k, v, ks, vs, table, starts, lengths)
    assert np.isnan(got).all()


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (32, 8, 128), (6, 6, 80), (8, 1, 256), (40, 1, 48)])
@pytest.mark.parametrize("cached,fresh,gain", [([0] * 6, [1] * 6, 1.0), ([1, 2, 3, 5, 9], [1, 1, 1, 2, 1], 2.0), ([700, 90, 3000], [1, 2, 1], 4.0)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_results_of_few_tokens_are_rounded_once(dtype, heads, kv_heads, d, cached, fresh, gain):
    """No weight is rounded to as few bits as the result.

    The bound is that of the other tests without a weight's 2^-11.  In its place: a weight's second part, 2^-11 of it at most, is off by 2^-11 of itself, 2^-22.
    """
    from meganeura_b200 import ops
    rng = np.random.default_rng(heads * d + len(cached))
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, 16, cached, fresh, gain=gain)
    args = [*(dev(x) for x in (k, v, ks, vs)), *(words(x) for x in (table, starts, lengths)), max(fresh)]
    got = host(ops.paged_attention_int8(q, *args))
    want, size, reach = PO.attention(host(q), IO.values(k, ks), IO.values(v, vs), table, starts, lengths, d ** -0.5)
    bound = attention_bound(dtype, want, size, reach, d, int(max(lengths)) * 127.0 * vs.max()) + (2.0 ** -22 - 2.0 ** -11) * size
    off = np.abs(got - want)
    assert (off <= bound).all(), f"off by {off.max():.3g}, {(off / bound).max():.2f} times the bound"


def exact_scale(exponent):
    """An f32 whose product with log2(e), as f32 rounds it, is 2^exponent."""
    log2e, x = np.float32(1.4426950408889634), np.float32(2.0 ** exponent / 1.4426950408889634)
    for _ in range(8):
        if x * log2e == np.float32(2.0 ** exponent):
            return float(x)
        x = np.nextafter(x, np.float32(np.inf) if x * log2e < 2.0 ** exponent else np.float32(0))
    raise AssertionError("no such number")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("cached,largest,others", [(60, 40, [3, 7, 50]), (300, 200, [3, 190, 260]), (300, 2, [130, 131, 299]), (5000, 4000, [10, 3000, 4500])])
@pytest.mark.parametrize("fresh", [1, 60])
def test_what_huge_scores_may_lose(dtype, cached, largest, others, fresh):
    """Scores beyond 2^20 whose largest belongs to a value of zeros: weights of 2^-22, 2^-24 and 2^-26 of it are all that is left.

    Every score is exact: its exponent is 2^14 (c0 + c1 2^-13) for a key's first two codes.  Weights and scales are powers of two, so that only what the operator says may be
    lost: 2^-29 of the largest weight times the largest scale, for the three keys that have a weight, a code being 127 at most; and the result's rounding, 2^-20 for the f32 sums.
    """
    from meganeura_b200 import ops
    rng = np.random.default_rng(cached)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, dtype, 2, 1, 64, 16, 16, [cached], [fresh])
    q[:] = 0
    q[..., 0], q[..., 1] = 1, 2.0 ** -13
    k[:], ks[:], vs[:] = 0, 1, 4
    at = lambda i: (table[0, i // 16], i % 16)
    k[at(largest)][:, 0] = 100
    v[at(largest)] = 0
    want = np.zeros(64)
    for i, key in enumerate(others):
        k[at(key)][:, :2] = 100, -11 - i
        want += 4.0 * v[at(key)][0] * 2.0 ** (-22 - 2 * i)
    bound = (EPS[dtype] / 2 + 2.0 ** -20) * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0) + 3 * 2.0 ** -29 * 127 * 4
    caches = [dev(x) for x in (k, v, ks, vs)]
    for t in (table, wider(table, 16, 2 ** 15), wider(table, 16, 2 ** 20)):      # which kernels serve it depends on how far the table reaches
        got = host(ops.paged_attention_int8(q, *caches, *(words(x) for x in (t, starts, lengths)), fresh, scale=exact_scale(14)))
        off = np.abs(got - want)
        assert (off <= bound).all(), f"off by {off.max():.3g}, {(off / bound).max():.2f} times the bound"
    # beside rows whose scores are small
    q[::2, 0, 0] = 2.0 ** -14
    check_attention(dtype, q, k, v, ks, vs, table, starts, lengths, scale=exact_scale(14))


@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 64), (4, 2, 128), (6, 3, 64), (8, 1, 256)])
@pytest.mark.parametrize("most", [2 ** 29, 2 ** 30, 2 ** 31, 2 ** 32 - 1])
def test_a_bound_of_new_tokens_that_is_far_too_large(heads, kv_heads, d, most):
    """Times the heads of a unit it passes 32 bits; rows off 16 bytes, so that the kernel of few tokens takes the call."""
    import torch
    rng = np.random.default_rng(d)
    q, k, v, ks, vs, *rest = attention_inputs(rng, "bf16", heads, kv_heads, d, 32, 16, [900, 40], [5, 1])
    wide = torch.zeros(q.shape[0], heads * d + 3, dtype=q.dtype, device="cuda")
    view = wide[:, 1:1 + heads * d].unflatten(1, (heads, d))
    view.copy_(q)
    check_attention("bf16", view, k, v, ks, vs, *rest, out=torch.zeros_like(wide)[:, 1:1 + heads * d].unflatten(1, (heads, d)), most=most)


def orders(rng, rows):
    """Ways in which a step's rows may stand: mixed, from the last to the first, as every seventh, one behind another but for the first, with pauses."""
    yield rng.permutation(rows)
    yield np.arange(rows)[::-1]
    yield np.argsort(np.arange(rows) % 7, kind="stable")
    yield np.roll(np.arange(rows), -1)
    yield np.insert(np.arange(rows), np.sort(rng.integers(0, rows + 1, rows // 3 + 1)), -1)


@pytest.mark.parametrize("kv_heads,d,page,block,cached,fresh", [
    (2, 64, 16, 16, [3], [2]),
    (2, 64, 32, 16, [0, 15, 40, 7, 16], [40, 1, 33, 2, 16]),
    (8, 128, 64, 64, [10, 0, 63, 100], [300, 64, 1, 500]),
    (1, 256, 32, 16, [5, 0], [700, 90]),
    (3, 16, 1024, 1024, [0, 1000, 20], [1500, 30, 900]),
    (2, 48, 256, 128, [1] * 50, [3] * 50),
    (2, 32, 16, 16, [9] * 1500, [2] * 1500),
])
def test_append_of_rows_in_any_order(kv_heads, d, page, block, cached, fresh):
    """Codes and scales are those of the rows in order, and the restatement's, wherever the rows of a block stand."""
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(d * page + len(cached))
    total = np.asarray(cached) + np.asarray(fresh)
    pages = int(sum(-(-n // page) for n in total)) + 2
    table = block_table(rng, total, page, pages)
    slots = np.concatenate([table[s, np.arange(c, c + n) // page] * page + np.arange(c, c + n) % page for s, (c, n) in enumerate(zip(cached, fresh))])
    positions, rows = np.concatenate([np.arange(c, c + n) for c, n in zip(cached, fresh)]), len(slots)
    x = (rng.standard_normal((2, rows, kv_heads, d)) * np.exp(rng.standard_normal((1, rows, 1, 1)))).astype(np.float32)
    before = [cache_of(rng, pages, page, block, kv_heads, d) for _ in range(2)]

    def append(order, theta, skip=0):
        at, spare = np.where(order < 0, 0, order), [-1] * skip
        c, s = [dev(b[0]) for b in before], [dev(b[1]) for b in before]
        ops.paged_append_int8(None, dev(x[0, at]), dev(x[1, at]), words(positions[at]), words([*spare, *np.where(order < 0, -1, slots[at])])[skip:], *c,
                              *s, theta=theta)
        return [host(t) for t in (*c, *s)]

    want = [IO.append(*b, y, slots) for b, y in zip(before, x)]
    rotated = append(np.arange(rows), 1e4)
    for order in orders(rng, rows):
        got = append(order, 0.0)
        for i in range(2):
            assert np.array_equal(got[i], want[i][0]) and np.array_equal(got[2 + i], want[i][1])
        assert all(np.array_equal(a, b) for a, b in zip(append(order, 1e4, skip=1), rotated))          # slots off 16 bytes, too


def test_no_wait_ran_out():
    from meganeura_b200 import ops
    ops.device_status()
