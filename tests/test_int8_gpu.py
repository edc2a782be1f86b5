"""The operators of 8-bit integers on a B200, each against its plain restatement in 64 bits, and a serving loop of them together."""
import numpy as np
import pytest

from int8_util import attention_inputs, cache_of, check_attention
from oracle import int8_oracle as IO
from oracle import paged_oracle as PO
from paged_util import EPS, host, torch_type, words

pytestmark = pytest.mark.gpu


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


# ---------------------------------------------------------------------------------------------- rows of codes

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k,more,skip", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 64, 0, 0), (2, 4096, 16, 8), (9, 1000, 0, 0), (4, 1001, 3, 1), (1, 16384, 0, 0), (2, 16392, 8, 0),
                                               (2, 40000, 0, 0), (300, 96, 0, 0), (2, 2056, 0, 4)])
def test_quantize_rows(dtype, rows, k, more, skip):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(rows * k)
    x = (rng.standard_normal((rows, k + more + skip)) * np.exp2(rng.integers(-12, 12, (rows, 1)))).astype(np.float32)
    x = torch.from_numpy(x).cuda().to(torch_type(dtype))[:, skip:skip + k]
    codes, scales = ops.quantize_rows(x)
    want, want_scales = IO.quantize_rows(host(x))
    assert np.array_equal(host(scales), want_scales) and np.array_equal(host(codes), want)


def test_quantize_rows_that_are_zero_tiny_huge_or_not_finite():
    from meganeura_b200 import ops
    x = np.random.default_rng(2).standard_normal((9, 200)).astype(np.float32)
    x[0], x[2] = 0, x[2] * np.float32(1e-32)
    x[3] *= np.float32(2e37)
    x[4, 199], x[5, 0], x[6, 7] = np.nan, np.inf, -np.inf
    x[7] = np.float32(2.0 ** -100)
    x[8, :2] = 127, 0.5                                  # a tie goes to the even code
    codes, scales = (host(t) for t in ops.quantize_rows(dev(x)))
    want, want_scales = IO.quantize_rows(x)
    assert np.array_equal(codes, want) and np.array_equal(scales, want_scales, equal_nan=True)
    assert scales[2] == 0 and scales[7] > 0 and np.isnan(scales[4]) and np.isinf(scales[5:7]).all() and codes[8, 1] == 0


def test_codes_and_scales_are_those_of_the_formulas_in_torch():
    """On the GPU, where torch divides by a number with a product: a large product of f32 rows may not show a code that fell to the other side of a tie."""
    import torch
    from meganeura_b200 import ops
    x = torch.randn(2000, 4096, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    codes, scales = ops.quantize_rows(x)
    scale = x.abs().amax(1) / 127
    assert torch.equal(scales, scale)
    assert torch.equal(codes.float(), (x * (1 / scale)[:, None]).round())


# ---------------------------------------------------------------------------------------------- products

def product_bound(dtype, want, addend):
    """The sum is a whole number; as f32, times two scales, plus the addend: four roundings of 2^-24, then the type's (2^-25 where f16 is subnormal)."""
    size = np.abs(want) + (0 if addend is None else 2 * np.abs(addend))
    return EPS[dtype] / 2 * np.abs(want) * 1.01 + 5 * 2.0 ** -24 * size + (2.0 ** -25 if dtype == "f16" else 1e-30)


def check_product(rng, dtype, m, k, n, with_addend=False, pitch=0, extreme=False):
    import torch
    from meganeura_b200 import ops
    a, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((m, k), (n, k)))
    if extreme:
        a[:], w[:] = -128, np.where(np.arange(n)[:, None] % 2, 127, -128)
    sa, sw = (rng.random(s).astype(np.float32) + 0.01 for s in (m, n))
    if dtype == "f16":                                   # sums of k products of up to 127^2 within its range
        sa *= np.float32(2.0 ** -8)
    t = torch_type(dtype)
    addend = torch.from_numpy(rng.standard_normal((m, n)).astype(np.float32) * 100 * k ** 0.5).cuda().to(t) if with_addend else None
    buffer = torch.full((m + 2, n + pitch), 7.0, dtype=t, device="cuda")
    out = buffer[1:m + 1, :n] if pitch or m > 1 else buffer[1:2, :n]
    got = host(ops.matmul_int8(dev(a), dev(sa), dev(w), dev(sw), addend=addend, out=out))
    add = None if addend is None else host(addend).astype(np.float64)
    want = IO.matmul(a, sa, w, sw, add)
    off, bound = np.abs(got - want), product_bound(dtype, want, add)
    assert (off <= bound).all(), f"off by {off.max():.3g}, {(off / bound).max():.2f} times the bound"
    buffer[1:m + 1, :n] = 7.0
    assert (buffer == 7.0).all()                         # nothing beside the result was written


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 16, 1), (1, 576, 1536), (2, 48, 17), (3, 4096, 100), (7, 1008, 33), (8, 64, 16), (8, 4096, 300), (9, 128, 40), (15, 2064, 129), (16, 512, 64)])
def test_product_of_few_rows(dtype, m, k, n):
    check_product(np.random.default_rng(m * k * n), dtype, m, k, n, with_addend=bool(n % 2), pitch=n % 3)


@pytest.mark.parametrize("m,k,n", [(8, 1040, 2380), (3, 80, 2369), (8, 576, 7001), (5, 1104, 7120), (1, 4096, 2368), (8, 1024, 2368)])
def test_product_of_few_rows_by_many_columns(m, k, n):
    check_product(np.random.default_rng(m * k * n), "bf16", m, k, n)


@pytest.mark.parametrize("m,k,n", [(17, 64, 31), (33, 160, 65), (64, 4096, 200), (100, 1536, 130), (128, 128, 128), (129, 144, 257), (203, 1536, 300), (255, 2048, 127), (257, 528, 640),
                                   (300, 16, 300), (700, 1040, 90)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_product_of_many_rows(dtype, m, k, n):
    check_product(np.random.default_rng(m * k * n), dtype, m, k, n, with_addend=bool(m % 2), pitch=m % 5)


@pytest.mark.parametrize("m,k,n", [(2048, 144, 10240), (1900, 80, 10000), (600, 64, 19456), (300, 96, 19100)])
def test_product_of_more_tiles_than_fit_at_once(m, k, n):
    """Several rounds of tiles, the last of them cut."""
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(m)
    a, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((m, k), (n, k)))
    sa, sw = (rng.random(s).astype(np.float32) + 0.01 for s in (m, n))
    got = host(ops.matmul_int8(dev(a), dev(sa), dev(w), dev(sw), dtype=torch.float32))
    for rows in np.array_split(np.arange(m), 8):
        want = IO.matmul(a[rows], sa[rows], w, sw)
        assert (np.abs(got[rows] - want) <= product_bound("f32", want, None)).all()


@pytest.mark.parametrize("m,k,n", [(128, 5120, 700), (300, 5120, 1000), (500, 5120, 1000), (700, 5120, 900), (1000, 5120, 1000), (1000, 5120, 1100), (1500, 2064, 100), (90, 4096, 1600),
                                   (150, 64, 20000), (250, 64, 29000), (600, 528, 6000), (600, 336, 4000), (48, 64, 40000), (10, 32, 40000), (96, 144, 38016), (64, 48, 38100), (100, 5120, 9000)])
def test_product_of_every_width_and_split(m, k, n):
    check_product(np.random.default_rng(m * k + n), "bf16", m, k, n, with_addend=bool(n % 200))


@pytest.mark.parametrize("m", [1, 9, 40, 300])
def test_product_at_the_largest_k(m):
    check_product(np.random.default_rng(m), "f32", m, 131056, 70, extreme=True)


def test_product_of_views_and_the_addend_in_place():
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(5)
    for m in (3, 50):
        a, w = (rng.integers(-127, 128, s).astype(np.int8) for s in ((m, 256), (90, 256)))
        sa, sw = (rng.random(s).astype(np.float32) for s in (m, 90))
        wide = torch.randn(m, 200, device="cuda")
        out = wide[:, 5:95]
        want = IO.matmul(a, sa, w, sw, host(out).astype(np.float64))
        before = host(wide).copy()
        assert ops.matmul_int8(dev(a), dev(sa), dev(w), dev(sw), addend=out, out=out) is out
        assert (np.abs(host(out) - want) <= product_bound("f32", want, before[:, 5:95])).all()
        assert np.array_equal(host(wide)[:, :5], before[:, :5]) and np.array_equal(host(wide)[:, 95:], before[:, 95:])


def test_rows_that_are_not_finite_stay_in_their_row():
    import torch
    from meganeura_b200 import ops
    for m in (6, 70):
        x, w = torch.randn(m, 512, device="cuda"), torch.randn(100, 512, device="cuda")
        x[2, 9], w[7, 1] = float("nan"), float("inf")
        y = host(ops.matmul_int8(*ops.quantize_rows(x), *ops.quantize_rows(w), dtype=torch.float32))
        bad = np.zeros_like(y, bool)
        bad[2], bad[:, 7] = True, True
        assert np.array_equal(np.isnan(y), bad)


# ---------------------------------------------------------------------------------------------- new keys and values

def check_append(rng, src, dtype, heads, kv_heads, d, page, block, cached, fresh, pad=0, theta=1e6, strided=True):
    """A step of sequences with `cached` tokens: caches and queries against the restatement, block by block."""
    import torch
    from meganeura_b200 import ops
    total = np.asarray(cached) + np.asarray(fresh)
    pages = int(sum(-(-n // page) for n in total)) + 2
    order, at, slots, positions = rng.permutation(pages), 0, [], []
    for c, n in zip(cached, fresh):
        need = -(-(c + n) // page)
        mine = order[at:at + need]
        at += need
        slots += [int(mine[i // page]) * page + i % page for i in range(c, c + n)]
        positions += range(c, c + n)
    slots, positions = np.array(slots + [-1] * pad), np.array(positions + [0] * pad)
    rows = len(slots)
    codes, scales = zip(*(cache_of(rng, pages, page, block, kv_heads, d) for _ in range(2)))
    codes, scales = [c.copy() for c in codes], [s.copy() for s in scales]
    t, wide = torch_type(src), (heads + 2 * kv_heads) * d + (3 if strided else 0)
    qkv = torch.from_numpy(rng.standard_normal((rows, wide)).astype(np.float32)).cuda().to(t)
    q, k, v = (qkv[:, a:b].unflatten(1, (-1, d)) for a, b in ((0, heads * d), (heads * d, (heads + kv_heads) * d), ((heads + kv_heads) * d, (heads + 2 * kv_heads) * d)))
    c, s = [dev(x) for x in codes], [dev(x) for x in scales]
    out = ops.paged_append_int8(q, k, v, words(positions), words(slots), *c, *s, theta=theta, q_dtype=torch_type(dtype))
    want = PO.rotate(host(q), positions, theta) if theta else host(q).astype(np.float64)
    assert out.dtype is torch_type(dtype)
    # angles of up to a turn in f32 and sines of them: 2^-22 of the pair's size each way, three roundings, then the type's
    pair = np.abs(host(q)).astype(np.float64)
    pair = np.concatenate([pair[..., :d // 2] + pair[..., d // 2:]] * 2, 2)
    assert (np.abs(host(out) - want) <= EPS[dtype] / 2 * np.abs(want) * 1.01 + 2.0 ** -20 * pair).all()
    for i, (x, rotated) in enumerate(((host(k), theta), (host(v), 0))):
        exact = (PO.rotate(x, positions, theta) if rotated else x).astype(np.float32)
        want_codes, want_scales = IO.append(codes[i], scales[i], exact, slots)
        got_codes, got_scales = host(c[i]), host(s[i])
        if not rotated:
            assert np.array_equal(got_scales, want_scales) and np.array_equal(got_codes, want_codes)
            continue
        # a rotated value is off by 2^-20 of its block's largest at most: the scale, too, and a value next to the border of two codes gets the other
        assert (np.abs(got_scales - want_scales) <= 2.0 ** -20 * want_scales).all()
        assert np.abs(got_codes.astype(int) - want_codes).max() <= 1 and (got_codes != want_codes).mean() <= 4 * 127 * 2.0 ** -20 + 2 / got_codes.size
        touched = np.zeros(pages * page // block, bool)
        touched[slots[slots >= 0] // block] = True
        same = ~np.repeat(touched, block).reshape(pages, page)
        assert np.array_equal(got_codes[same], codes[i][same])


@pytest.mark.parametrize("src,dtype", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,d,page,block,cached,fresh,pad", [
    (9, 3, 64, 16, 16, [0, 15, 16, 31, 100], [1, 1, 1, 1, 1], 0),
    (4, 2, 128, 64, 64, [0, 40, 63, 64, 5], [70, 1, 3, 64, 0], 3),
    (4, 1, 256, 32, 16, [7, 90], [50, 2], 1),
    (12, 12, 80, 128, 32, [100, 0, 33], [200, 5, 31], 40),
    (2, 2, 16, 1024, 1024, [0, 1000], [1500, 30], 0),
    (1, 1, 48, 256, 128, [1], [300], 0),
])
def test_append(src, dtype, heads, kv_heads, d, page, block, cached, fresh, pad):
    check_append(np.random.default_rng(d * page + len(cached)), src, dtype, heads, kv_heads, d, page, block, cached, fresh, pad)


def test_append_of_many_rows_takes_windows_of_rows():
    check_append(np.random.default_rng(9), "bf16", "bf16", 4, 2, 64, 32, 32, [3, 0, 17] + [9] * 40, [900, 700, 33] + [3] * 40, 7, strided=False)


def test_append_token_by_token_and_blocks_that_grow():
    from meganeura_b200 import ops
    rng = np.random.default_rng(11)
    codes, scales = cache_of(rng, 4, 32, 16, 2, 64)
    scales[:] = np.nan                                   # pages as they were left: a block's first token starts it anew
    c, s = dev(codes), dev(scales)
    other = [dev(codes), dev(scales)]
    for r in range(70):
        x = (rng.standard_normal((1, 2, 64)) * (30 if r in (5, 40) else 1)).astype(np.float32)
        slot = np.array([2, 0, 3])[r // 32] * 32 + r % 32
        codes, scales = IO.append(codes, scales, x, [slot])
        ops.paged_append_int8(None, dev(x), dev(x), words([r]), words([slot]), c, other[0], s, other[1])
        assert np.array_equal(host(s), scales, equal_nan=True) and np.array_equal(host(c), codes), r
        assert np.array_equal(host(other[0]), codes)


def test_append_of_values_that_are_not_finite_and_of_zeros():
    from meganeura_b200 import ops
    rng = np.random.default_rng(12)
    codes, scales = cache_of(rng, 3, 32, 16, 2, 32)
    x = rng.standard_normal((40, 2, 32)).astype(np.float32)
    x[3, 0, 5], x[20, 1, 0], x[32:] = np.nan, np.inf, 0
    slots = np.concatenate([np.arange(32) + 33, [0, 1, 2, 3], [17, 18, 96, -1]])       # the last block is not anew; a slot behind the cache is not written
    want = IO.append(codes, scales, x, slots)
    c, s, c2, s2 = (dev(t) for t in (codes, scales, codes, scales))
    ops.paged_append_int8(None, dev(x), dev(x), words(np.arange(40)), words(slots), c, c2, s, s2)
    assert np.array_equal(host(s), want[1], equal_nan=True) and np.array_equal(host(c), want[0]) and np.array_equal(host(c2), want[0])
    assert np.isnan(host(s)[1, 0, 0]) and host(s)[0, 0, 0] == 0


# ---------------------------------------------------------------------------------------------- attention

HEADS = [(9, 3, 64), (8, 2, 128), (6, 6, 80), (8, 1, 128), (14, 2, 64), (8, 1, 256), (3, 1, 16), (40, 1, 48), (2, 2, 192)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32), (256, 128)])
def test_attention_of_single_tokens(dtype, heads, kv_heads, d, page, block):
    rng = np.random.default_rng(heads * d + page)
    cached = [0, 1, 15, 16, 17, 31, 127, 128, 129, 700]
    check_attention(dtype, *attention_inputs(rng, dtype, heads, kv_heads, d, page, block, cached, [1] * len(cached), gain=2.0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("window", [0, 1, 17, 200])
def test_attention_of_a_few_tokens(dtype, heads, kv_heads, d, window):
    rng = np.random.default_rng(heads * d + window)
    check_attention(dtype, *attention_inputs(rng, dtype, heads, kv_heads, d, 32, 16, [0, 300, 5, 129, 40, 0], [3, 5, 0, 2, 1, 0], rows=14), window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("cached,fresh,page,block,window", [([0], [130], 64, 64, 0), ([200, 0, 33], [70, 1, 129], 16, 16, 0), ([500, 3], [40, 200], 128, 32, 100),
                                                            ([64, 0, 1000], [300, 0, 2], 32, 16, 33)])
def test_attention_of_many_tokens(dtype, heads, kv_heads, d, cached, fresh, page, block, window):
    rng = np.random.default_rng(heads * d + page)
    check_attention(dtype, *attention_inputs(rng, dtype, heads, kv_heads, d, page, block, cached, fresh, rows=sum(fresh) + 5, gain=1.5), window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", HEADS)
@pytest.mark.parametrize("cached,fresh,width,window", [([200, 0, 33, 700, 1, 90], [70, 1, 129, 2, 0, 40], 0, 0), ([700, 5, 40], [1, 100, 3], 1100, 150)])
def test_attention_of_many_tokens_beside_few(dtype, heads, kv_heads, d, cached, fresh, width, window):
    """More than four sequences, and tables that reach far: the sequences of few tokens have a launch of their own."""
    rng = np.random.default_rng(heads * d)
    q, k, v, ks, vs, table, *rest = attention_inputs(rng, dtype, heads, kv_heads, d, 16, 16, cached, fresh, rows=sum(fresh) + 5, gain=1.5)
    if width:
        table = np.concatenate([table, np.full((len(table), width - table.shape[1]), -1, table.dtype)], 1)
    check_attention(dtype, q, k, v, ks, vs, table, *rest, window=window)


@pytest.mark.parametrize("fresh", [1, 3, 150])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_of_scales_that_differ_widely(dtype, fresh):
    rng = np.random.default_rng(fresh)
    q, k, v, ks, vs, *rest = attention_inputs(rng, dtype, 8, 2, 64, 32, 16, [700, 90], [fresh, fresh], spread=0.2)
    vs *= np.exp2(rng.integers(-14, 14, vs.shape)).astype(np.float32)
    vs[rng.random(vs.shape) < 0.2] = 0
    ks[rng.random(ks.shape) < 0.2] = 0
    check_attention(dtype, q, k, v, ks, vs, *rest)
    check_attention(dtype, q, k, v, ks, np.zeros_like(vs), *rest)
    check_attention(dtype, q, k, v, ks, vs * np.float32(2.0 ** 60), *rest) if dtype == "bf16" else None


@pytest.mark.parametrize("fresh", [1, 5, 150])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_of_scales_that_nobody_sees(dtype, fresh):
    """Pages that nobody holds, places behind a sequence's end and blocks in front of a window may hold any scale; one that is seen makes its rows NaN."""
    rng = np.random.default_rng(fresh)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, dtype, 8, 2, 64, 64, 16, [600, 0], [fresh, fresh])
    held = np.zeros((*vs.shape[:2],), bool)
    for s, n in enumerate(lengths):
        for i in range(-(-int(n) // 16)):
            if s == 1 or i * 16 + 16 > n - fresh + 1 - 100:
                held[table[s, i * 16 // 64], i % 4] = True
    for x in (ks, vs):
        x[~held] = np.where(rng.random(x[~held].shape) < 0.5, np.nan, np.inf)
    got = check_attention(dtype, q, k, v, ks, vs, table, starts, lengths, window=100)
    assert np.isfinite(got).all()
    if fresh > 40:                                       # a block that only the later rows of a tile see
        for x in (ks, vs):
            y = x.copy()
            y[table[1, 32 // 64], 32 // 16 % 4, 0] = np.nan
            got = check_attention(dtype, q, k, v, y if x is ks else ks, y if x is vs else vs, table, starts, lengths, window=100)
            assert np.isnan(got).any()


@pytest.mark.parametrize("fresh", [1, 40])
def test_attention_over_pages_that_do_not_exist(fresh):
    rng = np.random.default_rng(fresh)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, "bf16", 4, 2, 128, 32, 16, [300, 200, 0], [fresh, fresh, fresh])
    table[0, 2], table[1, :] = -1, 10 ** 6
    check_attention("bf16", q, k, v, ks, vs, table, starts, lengths)


@pytest.mark.parametrize("fresh", [1, 60])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-6, 30.0])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_of_any_scale(dtype, fresh, scale):
    rng = np.random.default_rng(3)
    check_attention(dtype, *attention_inputs(rng, dtype, 4, 2, 64, 16, 16, [250, 3], [fresh, fresh], gain=0.3), scale=scale)


@pytest.mark.parametrize("fresh", [1, 60])
@pytest.mark.parametrize("gain", [2.0 ** -60, 2.0 ** 60, 2.0 ** 100])
def test_attention_of_queries_beyond_f16(fresh, gain):
    rng = np.random.default_rng(4)
    q, k, v, ks, vs, *rest = attention_inputs(rng, "bf16", 4, 2, 64, 16, 16, [250, 3], [fresh, fresh])
    check_attention("bf16", q * gain, k, v, ks, vs, *rest, scale=0.2 / gain)


@pytest.mark.parametrize("fresh", [1, 60])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 22, 2.0 ** 30, 2.0 ** 40])
def test_attention_of_huge_scores(fresh, size):
    """One key stands out by far more than the scores' precision: the result is its value, whatever the scores' size."""
    rng = np.random.default_rng(6)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, "f16", 2, 1, 64, 16, 16, [250], [fresh])
    q[:] = 1.0
    k[:] = rng.integers(-3, 4, k.shape)
    at = 100
    k[table[0, at // 16], at % 16] = 100
    ks[:] = 1 / 64
    got = check_attention("f16", q, k, v, ks, vs, table, starts, lengths, scale=size)
    want = v[table[0, at // 16], at % 16, 0] * vs[table[0, at // 16], 0, 0]
    assert (np.abs(got - want) <= 2.0 ** -10 * np.abs(want)).all()


@pytest.mark.parametrize("fresh", [1, 4, 90])
def test_attention_of_strided_and_misaligned_rows(fresh):
    import torch
    rng = np.random.default_rng(7)
    q, k, v, ks, vs, *rest = attention_inputs(rng, "bf16", 6, 2, 64, 32, 32, [70, 9], [fresh, fresh])
    for skip, more in ((8, 64), (1, 3)):
        wide = torch.zeros(q.shape[0], 6 * 64 + skip + more, dtype=q.dtype, device="cuda")
        view = wide[:, skip:skip + 6 * 64].unflatten(1, (6, 64))
        view.copy_(q)
        out = torch.full_like(wide, 5.0)
        check_attention("bf16", view, k, v, ks, vs, *rest, out=out[:, skip:skip + 6 * 64].unflatten(1, (6, 64)))
        assert (out[:, :skip] == 5.0).all() and (out[:, skip + 6 * 64:] == 5.0).all()


def test_attention_of_more_new_tokens_than_was_said():
    rng = np.random.default_rng(8)
    check_attention("f16", *attention_inputs(rng, "f16", 8, 2, 64, 16, 16, [5, 300], [90, 70]), most=1)


@pytest.mark.parametrize("sequences,fresh", [(1, 1), (200, 1), (60, 4), (3, 400)])
def test_attention_is_the_same_from_run_to_run(sequences, fresh):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(sequences)
    q, k, v, ks, vs, table, starts, lengths = attention_inputs(rng, "bf16", 8, 2, 128, 64, 32, rng.integers(0, 900, sequences), [fresh] * sequences)
    args = [q, *(dev(x) for x in (k, v, ks, vs)), *(words(x) for x in (table, starts, lengths)), fresh]
    first = ops.paged_attention_int8(*args)
    for _ in range(3):
        assert torch.equal(ops.paged_attention_int8(*args), first)


# ---------------------------------------------------------------------------------------------- together

def test_a_layer_in_8_bits_captured_and_replayed():
    """Plan, projection, append, attention and output projection of steps of many sequences from one graph, against the same operators in 64 bits."""
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(21)
    S, H, KV, D, width, page, block, pages, rows = 5, 4, 2, 64, 256, 32, 16, 64, 48
    w_qkv, w_o = ((rng.standard_normal(s) * 0.1).astype(np.float32) for s in (((H + 2 * KV) * D, width), (width, H * D)))
    wq, wo = ops.quantize_rows(dev(w_qkv)), ops.quantize_rows(dev(w_o))
    k_cache, v_cache = (torch.zeros(pages, page, KV, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((pages, page // block, KV), float("nan"), device="cuda") for _ in range(2))
    cached, fresh, held = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(3))
    table = torch.full((S, 12), -1, dtype=torch.int32, device="cuda")
    free, count = words(rng.permutation(pages)), words([pages])
    x, step = torch.zeros(rows, width, device="cuda"), ops.PagedStep.empty(S, rows)
    y = torch.zeros(rows, width, device="cuda")

    def layer():
        ops.paged_plan(cached, fresh, table, held, free, count, page, rows, step=step)
        qkv = ops.matmul_int8(*ops.quantize_rows(x), *wq, dtype=torch.bfloat16)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, KV * D, KV * D], 1))
        q = ops.paged_append_int8(q, k, v, step.positions, step.slots, k_cache, v_cache, ks, vs, theta=1e4)
        o = ops.paged_attention_int8(q, k_cache, v_cache, ks, vs, table, step.starts, step.lengths, 20)
        ops.matmul_int8(*ops.quantize_rows(o.flatten(1)), *wo, addend=x, out=y)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer()                                          # nothing is fresh yet
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    lengths = np.zeros(S, int)
    history = [np.zeros((0, KV, D))] * S, [np.zeros((0, KV, D))] * S
    for now in ([20, 3, 0, 7, 9], [1, 1, 20, 1, 5], [1, 0, 1, 2, 1], [3, 1, 1, 1, 1]):
        data = rng.standard_normal((rows, width)).astype(np.float32)
        x.copy_(torch.from_numpy(data))
        cached.copy_(words(lengths))
        fresh.copy_(words(now))
        graph.replay()
        got = host(y)
        r = 0
        wq_values, wo_values = (host(c).astype(np.float64) * host(s)[:, None] for c, s in (wq, wo))
        for s, n in enumerate(now):
            if n == 0:
                continue
            a = data[r:r + n]
            codes, scales = IO.quantize_rows(a)
            qkv = (codes * scales[:, None].astype(np.float64)) @ wq_values.T
            q, k, v = (qkv[:, i:j].reshape(n, -1, D) for i, j in ((0, H * D), (H * D, (H + KV) * D), ((H + KV) * D, (H + 2 * KV) * D)))
            at = np.arange(lengths[s], lengths[s] + n)
            q, k = PO.rotate(q, at, 1e4), PO.rotate(k, at, 1e4)
            for h, new in zip(history, (k, v)):
                h[s] = np.concatenate([h[s], new])
            keys, values = (np.repeat(h[s], H // KV, 1) for h in history)
            score = np.einsum("nhd,lhd->nhl", q, keys) / D ** 0.5
            score[np.broadcast_to((np.arange(len(keys)) > at[:, None])[:, None], score.shape)] = -np.inf
            w = np.exp(score - score.max(2, keepdims=True))
            o = np.einsum("nhl,lhd->nhd", w / w.sum(2, keepdims=True), values).reshape(n, -1)
            want = o @ wo_values.T + a
            # 8 bits for keys, values and the attention's results: 1/254 of a block's largest value each, about 1% of a value; the projections' weights are the same
            assert np.linalg.norm(got[r:r + n] - want) <= 0.03 * np.linalg.norm(want - a)
            r += n
        lengths += now


def test_two_streams_and_a_stream_argument():
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(31)
    inputs = [attention_inputs(rng, "bf16", 8, 2, 128, 64, 32, [3000, 50, 700], [1, 2, 1]) for _ in range(2)]
    args = [[q, *(dev(x) for x in (k, v, ks, vs)), *(words(x) for x in rest), 2] for q, k, v, ks, vs, *rest in inputs]
    x, w = torch.randn(40, 1024, device="cuda"), ops.quantize_rows(torch.randn(500, 1024, device="cuda"))
    want = [ops.paged_attention_int8(*a) for a in args], ops.matmul_int8(*ops.quantize_rows(x), *w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            got[i].append((ops.paged_attention_int8(*args[i], stream=s), ops.matmul_int8(*ops.quantize_rows(x, stream=s), *w, stream=s)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[0][i]) and torch.equal(y, want[1]) for o, y in got[i])


def test_python_refusals():
    import torch
    from meganeura_b200 import ops
    x = torch.randn(4, 64, device="cuda")
    codes, scales = ops.quantize_rows(x)
    for bad in (lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(x.t()), lambda: ops.quantize_rows(x, out=(codes, scales[:3])),
                lambda: ops.matmul_int8(codes, scales, codes[:, :32], scales), lambda: ops.matmul_int8(codes, scales, codes.t().contiguous().t(), scales),
                lambda: ops.matmul_int8(codes, scales[:2], codes, scales), lambda: ops.matmul_int8(codes, scales, codes, scales, dtype=torch.int8),
                lambda: ops.matmul_int8(codes, scales, codes, scales, out=x), lambda: ops.matmul_int8(codes, scales, codes, scales, addend=x[:, :4], dtype=torch.float16)):
        with pytest.raises(ValueError):
            bad()
    cache, s = torch.zeros(2, 32, 2, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, 2, device="cuda")
    k, w = torch.randn(1, 2, 64, device="cuda"), words([0])
    for bad in (lambda: ops.paged_append_int8(None, k, k, w, w, cache, cache, s, s[:, :1]), lambda: ops.paged_append_int8(None, k, k, w, w, cache, cache, s[:1], s[:1]),
                lambda: ops.paged_append_int8(None, k, k, w, w, cache.float(), cache, s, s), lambda: ops.paged_append_int8(None, k.double(), k.double(), w, w, cache, cache, s, s),
                lambda: ops.paged_append_int8(k.half(), k, k, w, w, cache, cache, s, s), lambda: ops.paged_append_int8(None, k, k[:, :1], w, w, cache, cache, s, s),
                lambda: ops.paged_append_int8(k, k, k, w, w, cache, cache, s, s, q_dtype=torch.float32),
                lambda: ops.paged_attention_int8(k, cache, cache, s, s, w[None], words([0, 1]), w, 1),
                lambda: ops.paged_attention_int8(k.half(), cache, cache, s, s, w[None], w, w, 1),
                lambda: ops.paged_attention_int8(k.half(), cache, cache, s, s, w[None], words([0, 1]), w, 0)):
        with pytest.raises(ValueError):
            bad()
