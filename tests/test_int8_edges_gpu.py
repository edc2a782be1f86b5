"""The 8-bit operators where they could go wrong: numbers beyond 32 bits, rows that are not finite, graphs replayed with other lengths, outputs in place."""
import numpy as np
import pytest

from int8_util import attention_bound, attention_inputs, cache_of, check_attention, wider
from oracle import int8_oracle as IO
from oracle import paged_oracle as PO
from paged_util import EPS, host, torch_type, words

pytestmark = pytest.mark.gpu


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


@pytest.mark.parametrize("fresh", [1, 60])
def test_a_cache_of_more_than_4_gib(fresh):
    """Pages at the end of caches of 4.5 GB: written by the append, read by the attention."""
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(fresh)
    kv, d, page, block, pages = 8, 128, 64, 32, 68000
    k, v = (torch.zeros(pages, page, kv, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, page // block, kv, device="cuda") for _ in range(2))
    assert k.numel() > 1 << 32
    held = [pages - 1, 3, pages - 2, pages - 5]
    length = 3 * page + 20
    table = np.full((1, 6), -1)
    table[0, :4] = held
    x = [torch.from_numpy(rng.standard_normal((length, kv, d)).astype(np.float32)).cuda() for _ in range(2)]
    slots = np.array([held[i // page] * page + i % page for i in range(length)])
    ops.paged_append_int8(None, *x, words(np.arange(length)), words(slots), k, v, ks, vs)
    small = np.zeros((4, page, kv, d), np.int8), np.zeros((4, page // block, kv), np.float32)
    codes, scales = zip(*(IO.append(*small, host(t), np.arange(length)) for t in x))
    for t, want in ((k, codes[0]), (v, codes[1])):
        assert np.array_equal(host(t[held]), want)
    for t, want in ((ks, scales[0]), (vs, scales[1])):
        assert np.array_equal(host(t[held]), want)
    q = torch.from_numpy(rng.standard_normal((fresh, 32, d)).astype(np.float32)).cuda().to(torch.bfloat16)
    want, size, reach = PO.attention(host(q), IO.values(codes[0], scales[0]), IO.values(codes[1], scales[1]), np.arange(4)[None], [0, fresh], [length], d ** -0.5)
    for t in (table, wider(table, page, 2 ** 20)):
        got = ops.paged_attention_int8(q, k, v, ks, vs, words(t), words([0, fresh]), words([length]), fresh)
        assert (np.abs(host(got) - want) <= attention_bound("bf16", want, size, reach, d, length * 5.0)).all()


def test_products_into_rows_that_are_far_apart():
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(1)
    buffer = torch.zeros(600, 1 << 23, dtype=torch.bfloat16, device="cuda")              # 10 GB: the last rows begin behind 2^32 elements
    a, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((600, 64), (50, 64)))
    sa, sw = (rng.random(s).astype(np.float32) for s in (600, 50))
    out = buffer[:, 7:57]
    want = IO.matmul(a, sa, w, sw)
    ops.matmul_int8(dev(a), dev(sa), dev(w), dev(sw), out=out)
    assert (np.abs(host(out) - want) <= EPS["bf16"] / 2 * np.abs(want) * 1.01 + 1e-6).all()
    assert float(buffer[:, 57:64].abs().max()) == 0 and float(buffer[:, :7].abs().max()) == 0
    x = buffer[:, 7:57].clone()
    codes, scales = ops.quantize_rows(out)
    again, scales_again = ops.quantize_rows(x)
    assert torch.equal(codes, again) and torch.equal(scales, scales_again)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("fresh,far", [(1, 0), (4, 0), (70, 0), (70, 2 ** 20), (70, 2 ** 14)])
def test_queries_that_are_not_finite_stay_in_their_head_and_row(dtype, fresh, far):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(fresh)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, dtype, 8, 2, 64, 16, 16, [300, 40], [fresh, fresh])
    table = wider(table, 16, far)
    args = [*(dev(x) for x in (k, v, ks, vs)), *(words(x) for x in (table, starts, lengths)), fresh]
    clean = host(ops.paged_attention_int8(q, *args))
    spoilt = q.clone()
    spoilt[0, 3] = float("nan")
    spoilt[fresh, 6, 5] = float("inf")
    got = host(ops.paged_attention_int8(spoilt, *args))
    bad = np.zeros(got.shape[:2], bool)
    bad[0, 3], bad[fresh, 6] = True, True
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(8, 2, 128), (9, 3, 64), (8, 1, 256)])
@pytest.mark.parametrize("fresh", [[1] * 6, [3, 1, 2, 5, 1, 4], [90, 1, 40, 3, 150, 33], [70, 65, 40, 33]])
def test_attention_of_rows_that_see_nothing_and_of_lengths_that_cannot_be(dtype, heads, kv_heads, d, fresh):
    """Sequences with fewer tokens than new ones, with none, longer than their table, and the last one's rows cut off behind the rows that are there."""
    rng = np.random.default_rng(heads * d + len(fresh))
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, 16, [200, 40, 0, 9, 64, 7][:len(fresh)], fresh)
    lengths[0], lengths[1], lengths[2] = 0, 10 ** 9, max(1, fresh[2] - 1)
    table[1, :] = np.arange(table.shape[1])
    starts[-1] += 50
    check_attention(dtype, q, k, v, ks, vs, table, starts, lengths, most=max(fresh))
    check_attention(dtype, q, k, v, ks, vs, table, starts, np.zeros_like(lengths), most=max(fresh))
    check_attention(dtype, q, k, v, ks, vs, table, starts, np.minimum(lengths, 30), most=max(fresh))


@pytest.mark.parametrize("heads,kv_heads,d,fresh", [(300, 1, 64, 1), (300, 1, 32, 5), (600, 2, 16, 2), (256, 1, 128, 3), (34, 2, 128, 2)])
def test_attention_of_very_many_heads_per_key_head(heads, kv_heads, d, fresh):
    rng = np.random.default_rng(heads + fresh)
    check_attention("bf16", *attention_inputs(rng, "bf16", heads, kv_heads, d, 32, 32, [300, 0, 31], [fresh] * 3))


@pytest.mark.parametrize("sequences", [1500, 4096])
def test_attention_of_very_many_sequences(sequences):
    rng = np.random.default_rng(sequences)
    fresh = rng.integers(0, 3, sequences)
    fresh[7] = 40
    check_attention("f16", *attention_inputs(rng, "f16", 4, 2, 64, 16, 16, rng.integers(0, 20, sequences), fresh, rows=int(fresh.sum()) + 3))


@pytest.mark.parametrize("most,far", [(2, 0), (40, 0), (40, 2 ** 13), (40, 2 ** 20)])
def test_a_captured_attention_follows_the_lengths(most, far):
    """One graph, replayed with sequences of other lengths and numbers of new tokens, beside another graph of the same operator."""
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(most)
    S, page, block, pages, rows = 4, 32, 16, 200, 4 * most
    k, ks = cache_of(rng, pages, page, block, 2, 64)
    v, vs = cache_of(rng, pages, page, block, 2, 64)
    d = [dev(x) for x in (k, v, ks, vs)]
    table = wider(rng.permutation(pages)[:S * 40].reshape(S, 40), page, far)
    q = torch.from_numpy(rng.standard_normal((rows, 8, 64)).astype(np.float32)).cuda().half()
    starts, lengths = words(np.zeros(S + 1)), words(np.zeros(S))
    outs = [torch.zeros_like(q) for _ in range(2)]
    graphs = []
    ops.paged_attention_int8(q, *d, words(table), starts, lengths, most, out=outs[0])
    t = words(table)
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.paged_attention_int8(q, *d, t, starts, lengths, most, out=out)
        graphs.append(g)
    for _ in range(4):
        fresh, cached = rng.integers(0, most + 1, S), rng.integers(0, 1000, S)
        at = np.concatenate([[0], np.cumsum(fresh)])
        starts.copy_(words(at))
        lengths.copy_(words(cached + fresh))
        for out, g in zip(outs, graphs):
            out.fill_(3.0)
            g.replay()
        want, size, reach = PO.attention(host(q), IO.values(k, ks), IO.values(v, vs), table, at, cached + fresh, 0.125)
        mine = np.arange(rows) < at[-1]
        for out in outs:
            got = host(out)
            assert (got[~mine] == 3.0).all()
            assert (np.abs(got - want)[mine] <= attention_bound("f16", want, size, reach, 64, 1100 * 10.0)[mine]).all()


def test_queries_rotated_in_place():
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(3)
    for rows in (1, 9, 300):
        q = torch.from_numpy(rng.standard_normal((rows, 6, 64)).astype(np.float32)).cuda().to(torch.bfloat16)
        k = torch.zeros(rows, 2, 64, dtype=torch.bfloat16, device="cuda")
        cache, scales = torch.zeros(12, 32, 2, 64, dtype=torch.int8, device="cuda"), torch.zeros(12, 1, 2, device="cuda")
        at = words(np.arange(rows) + 1000)
        args = (k, k, at, words(np.arange(rows)), cache, cache.clone(), scales, scales.clone())
        want = ops.paged_append_int8(q, *args, theta=1e4)
        got = ops.paged_append_int8(q, *args, theta=1e4, q_out=q)
        assert got is q and torch.equal(got, want)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_an_append_of_padded_rows_alone_changes_nothing(rows):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(rows)
    codes, scales = cache_of(rng, 3, 32, 16, 2, 64)
    x = torch.randn(rows, 2, 64, device="cuda")
    c, s = [dev(codes) for _ in range(2)], [dev(scales) for _ in range(2)]
    for slot in (-1, 96, 2 ** 31 - 1):
        ops.paged_append_int8(None, x, x, words(np.zeros(rows)), words(np.full(rows, slot)), *c, *s, theta=1e6)
    assert all(np.array_equal(host(t), codes) for t in c) and all(np.array_equal(host(t), scales) for t in s)


def test_drafts_that_were_taken_back_leave_the_tokens_in_front():
    """A block with a rejected draft of far larger values: what was in front keeps its value within the larger scale's half step, and the next token is right."""
    from meganeura_b200 import ops
    rng = np.random.default_rng(5)
    codes, scales = np.zeros((1, 32, 1, 64), np.int8), np.zeros((1, 1, 1), np.float32)
    x = rng.standard_normal((12, 1, 64)).astype(np.float32)
    x[9] *= 20                                           # the draft in slot 9
    c, s, c2, s2 = dev(codes), dev(scales), dev(codes), dev(scales)

    def put(rows, slots):
        ops.paged_append_int8(None, dev(x[rows]), dev(x[rows]), words(slots), words(slots), c, c2, s, s2)
    put(np.arange(8), np.arange(8))
    small = float(host(s)[0, 0, 0])
    put([8, 9], [8, 9])
    put([10], [9])                                       # slot 9 again, by the token that was taken instead
    large = float(host(s)[0, 0, 0])
    values = IO.values(host(c), host(s))[0, :, 0]
    assert large > 3 * small
    assert (np.abs(values[:8] - x[:8, 0]) <= 0.501 * (small + large)).all() and (np.abs(values[[8, 9]] - x[[8, 10], 0]) <= 0.501 * large).all()


def test_no_wait_ran_out():
    from meganeura_b200 import ops
    ops.device_status()
