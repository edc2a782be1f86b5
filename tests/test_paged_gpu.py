"""The operators over a paged cache on a B200, each against its plain restatement in 64 bits, and a serving loop of them together."""
import math

import numpy as np
import pytest

from oracle import paged_oracle as PO
from paged_util import EPS, attention_inputs, block_table, check_attention, host, torch_type, words

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- block tables and slots

def pool(rng, cached, page, pages, width):
    table = block_table(rng, cached, page, pages, width)
    held = np.array([-(-int(c) // page) for c in cached])
    used = set(table[table >= 0].tolist())
    free = np.full(pages, -1)
    left = [p for p in rng.permutation(pages) if p not in used]
    free[:len(left)] = left
    return table, held, free, len(left)


def check_plan(cached, fresh, table, held, free, count, page, rows):
    from meganeura_b200 import ops
    d = [words(x) for x in (cached, fresh, table, held, free, [count])]
    step = ops.paged_plan(*d, page, rows)
    starts, lengths, positions, slots, lacking, table1, held1, count1 = PO.plan(np.asarray(cached), np.asarray(fresh), table, held, free, count, page, rows)
    for name, have, want in (("starts", step.starts, starts), ("lengths", step.lengths, lengths), ("positions", step.positions, positions), ("slots", step.slots, slots),
                             ("lacking", step.lacking, [lacking]), ("table", d[2], table1), ("held", d[3], held1), ("count", d[5], [count1]), ("free", d[4], free)):
        assert np.array_equal(host(have), np.asarray(want)), name
    return d, step


@pytest.mark.parametrize("sequences,page,most,spare,rows_more", [
    (1, 8, 1, 4, 0), (1, 16, 900, 100, 3), (7, 16, 1, 0, 5), (8, 1024, 3, 8, 0), (33, 32, 70, 40, 1), (256, 16, 5, 64, 0), (700, 8, 9, 3000, 100), (1025, 16, 3, 900, 17),
    (4096, 8, 2, 5000, 1),
])
def test_plan_and_trim(sequences, page, most, spare, rows_more):
    from meganeura_b200 import ops
    rng = np.random.default_rng(sequences * 7 + page)
    cached, fresh = rng.integers(0, 5 * page, sequences), rng.integers(0, most + 1, sequences)
    width = -(-(5 * page + most) // page)
    pages = int(sum(-(-c // page) for c in cached)) + spare
    state = pool(rng, cached, page, pages, width)
    rows = max(1, int(fresh.sum()) + rows_more)
    d, step = check_plan(cached, fresh, *state, page, rows)
    # then some tokens are taken back
    keep = np.minimum(host(step.lengths), cached + rng.integers(0, most + 1, sequences))
    want = PO.trim(keep, host(d[2]), host(d[3]), host(d[4]), int(host(d[5])[0]), page)
    ops.paged_trim(words(keep), d[2], d[3], d[4], d[5], page)
    for have, w in zip((d[2], d[3], d[4], d[5]), want):
        assert np.array_equal(host(have), np.asarray(w).reshape(host(have).shape))
    # and everything
    ops.paged_trim(words(np.zeros(sequences)), d[2], d[3], d[4], d[5], page)
    assert int(host(d[5])[0]) == pages and (host(d[2]) == -1).all() and (host(d[3]) == 0).all()
    assert sorted(host(d[4]).tolist()) == list(range(pages))


def test_plan_when_pages_run_out_rows_run_out_or_a_row_of_the_table_is_too_narrow():
    rng = np.random.default_rng(5)
    # two pages free: the first need of one is served, the need of two is not, nor the one behind it; who needs none is
    check_plan([16, 10, 16, 3, 16], [1, 40, 1, 2, 16], *pool(rng, [16, 10, 16, 3, 16], 16, 7, 5), 16, 60)
    check_plan([16, 10], [100, 1], *pool(rng, [16, 10], 16, 20, 2), 16, 101)           # the first needs 8 pages in a table of 2
    check_plan([0, 0, 0], [9, 9, 9], *pool(rng, [0, 0, 0], 8, 9, 4), 8, 12)            # rows for the first and a part of the second
    check_plan([0, 5], [0, 0], *pool(rng, [0, 5], 8, 9, 4), 8, 3)
    table, held, free, count = pool(rng, [8, 8], 8, 6, 3)
    table[1, 0] = 77                                                                   # a page that does not exist has no slots
    check_plan([4, 4], [2, 6], table, held, free, count, 8, 8)
    check_plan([2 ** 31 - 9, 3], [4, 2 ** 31 - 1], *pool(rng, [0, 3], 8, 6, 3), 8, 8)   # lengths beyond any table
    # more pages held than needed: none are taken
    table, held, free, count = pool(rng, [30, 8], 8, 9, 5)
    check_plan([2, 8], [5, 1], table, held, free, count, 8, 6)


@pytest.mark.parametrize("sequences", [3, 300, 2000])
def test_plan_of_a_step_whose_lengths_are_the_next_steps_cached_tokens(sequences):
    from meganeura_b200 import ops
    rng, page, rows, steps = np.random.default_rng(sequences), 8, 3 * sequences, 4
    cached, pages, width = rng.integers(0, 20, sequences), 5 * sequences, 6
    table, held, free, count = pool(rng, cached, page, pages, width)
    step = ops.PagedStep.empty(sequences, rows)
    step.lengths.copy_(words(cached))
    d = [words(x) for x in (table, held, free, [count])]
    for _ in range(steps):                             # every one in the tensors of the one before
        fresh = rng.integers(0, 4, sequences)
        starts, lengths, positions, slots, lacking, table, held, count = PO.plan(cached, fresh, table, held, free, count, page, rows)
        ops.paged_plan(step.lengths, words(fresh), *d, page, rows, step=step)
        for name, want in (("starts", starts), ("lengths", lengths), ("positions", positions), ("slots", slots), ("lacking", [lacking])):
            assert np.array_equal(host(getattr(step, name)), np.asarray(want)), name
        assert np.array_equal(host(d[0]), table) and np.array_equal(host(d[1]), held) and host(d[3])[0] == count
        cached = lengths


# ---------------------------------------------------------------------------------------------- keys and values into the cache

@pytest.mark.parametrize("src,dtype", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows,heads,kv_heads,d,page,theta,layout", [
    (1, 9, 3, 64, 16, 1e4, "fused"), (5, 8, 2, 128, 8, 1e6, "fused"), (130, 4, 4, 80, 32, 5e5, "apart"), (3, 6, 1, 256, 64, 1e6, "odd"), (7, 5, 5, 6, 16, 1e4, "apart"),
    (4, 8, 2, 64, 16, 0.0, "fused"), (2500, 2, 1, 64, 16, 1e6, "fused"), (6, 0, 2, 128, 16, 1e6, "fused"),
])
def test_append(src, dtype, rows, heads, kv_heads, d, page, theta, layout):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(rows + d)
    pages = -(-rows // page) + 2
    pad = {"fused": 0, "apart": 24, "odd": 5}[layout]
    qkv = torch.from_numpy(rng.standard_normal((rows, (heads + 2 * kv_heads) * d + pad)).astype(np.float32)).cuda().to(torch_type(src))
    if layout == "odd":                                        # rows that begin anywhere
        qkv = torch.cat([qkv.flatten()[:1], qkv.flatten()])[1:].view(qkv.shape)
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv[:, :(heads + 2 * kv_heads) * d].split([heads * d, kv_heads * d, kv_heads * d], 1))
    caches = [torch.full((pages, page, kv_heads, d), 7.0, dtype=torch_type(dtype), device="cuda") for _ in range(2)]
    slots = rng.permutation(pages * page)[:rows]
    lost = rng.random(rows) < 0.2
    slots[lost] = rng.choice([-1, pages * page, 2 ** 31 - 1], lost.sum())
    positions = rng.integers(0, 10 if rows < 4 else 200000, rows)
    out = ops.paged_append(q if heads else None, k, v, words(positions), words(slots), *caches, theta=theta)
    turn = (lambda x: PO.rotate(host(x), positions, theta)) if theta else (lambda x: host(x).astype(np.float64))
    # a rotated value is two products and a sum of values that sine and cosine (2^-22 at most) and f32 leave 2^-21 of their size off; then one rounding
    def near(have, want, size):
        assert (np.abs(host(have) - want) <= EPS[dtype] / 2 * np.abs(want) + 2.0 ** -21 * size * bool(theta) + 2.0 ** -25 * (dtype == "f16")).all()
    reach = lambda x: np.concatenate([np.hypot(*np.split(np.abs(host(x).astype(np.float64)), 2, 2))] * 2, 2) * math.sqrt(2)  # noqa: E731
    if heads:
        assert out.dtype == torch_type(dtype) and out.shape == (rows, heads, d)
        near(out, turn(q), reach(q))
    else:
        assert out is None
    for cache, x, want, size in ((caches[0], k, turn(k), reach(k)), (caches[1], v, host(v).astype(np.float64), 0 * reach(v))):
        flat = cache.flatten(0, 1)
        near(flat[torch.from_numpy(slots[~lost]).cuda()], want[~lost], size[~lost])
        rest = np.setdiff1d(np.arange(pages * page), slots)
        assert (flat[torch.from_numpy(rest).cuda()] == 7.0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_rotates_queries_in_place(dtype):
    import torch
    from meganeura_b200 import ops
    q, k = (torch.randn(700, h, 64, device="cuda").to(torch_type(dtype)) for h in (6, 2))
    caches = [torch.zeros(90, 8, 2, 64, dtype=torch_type(dtype), device="cuda") for _ in range(2)]
    at = words(np.arange(700))
    want = ops.paged_append(q, k, k, at, at, *caches, theta=1e4)
    assert ops.paged_append(q, k, k, at, at, *caches, theta=1e4, q_out=q) is q and torch.equal(q, want)


def test_append_keeps_infinities_and_nan_as_a_cast_does():
    import torch
    from meganeura_b200 import ops
    x = torch.tensor([1e6, -1e6, float("inf"), float("nan"), 65519.0, 65520.0, 1e-9, -0.0], device="cuda").view(1, 1, 8)
    caches = [torch.zeros(1, 8, 1, 8, dtype=torch.float16, device="cuda") for _ in range(2)]
    ops.paged_append(None, x, x, words([0]), words([3]), *caches)
    for c in caches:
        assert torch.equal(c[0, 3, 0].view(torch.int16), x[0, 0].half().view(torch.int16))


# ---------------------------------------------------------------------------------------------- attention

SHAPES = [(9, 3, 64), (32, 8, 128), (4, 4, 80), (16, 2, 96), (8, 1, 128), (6, 2, 256), (3, 1, 20), (5, 5, 33), (40, 1, 64), (4, 2, 40), (2, 1, 8), (6, 3, 136)]
BATCHES = {
    "one": (16, [0], [1]), "two": (16, [1], [1]), "tile": (16, [31], [1]), "decode": (16, [5, 130, 0, 64, 63, 65, 700], [1] * 7),
    "drafts": (8, [3, 40, 257, 0], [5, 2, 4, 3]), "ragged": (32, [0, 77, 300, 12, 0], [40, 0, 3, 1, 129]), "chunk": (64, [200, 0], [150, 300]), "wide page": (1024, [900, 100], [9, 33]),
}


def run(q, k, v, table, starts, lengths, most, **kw):
    from meganeura_b200 import ops
    out = ops.paged_attention(q, k, v, words(table), words(starts), words(lengths), most, **kw)
    ops.device_status()                                            # no wait inside the kernels ran out
    return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,d", SHAPES)
@pytest.mark.parametrize("batch", BATCHES)
def test_attention(dtype, heads, kv_heads, d, batch):
    page, cached, fresh = BATCHES[batch]
    rng = np.random.default_rng(d + len(batch))
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, page, cached, fresh)
    got = run(q, k, v, table, starts, lengths, max(fresh))
    check_attention(dtype, q, k, v, table, starts, lengths, got, d ** -0.5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 17, 64, 128, 1000])
@pytest.mark.parametrize("heads,kv_heads,d", [(9, 3, 64), (8, 2, 128)])
def test_attention_in_a_window(dtype, window, heads, kv_heads, d):
    rng = np.random.default_rng(window)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 16, [300, 0, 129, 40], [1, 150, 5, 70])
    got = run(q, k, v, table, starts, lengths, 150, window=window, scale=0.3)
    check_attention(dtype, q, k, v, table, starts, lengths, got, 0.3, window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fresh", [[1, 1, 1, 1], [6, 1, 0, 4], [90, 30, 1, 60]])
def test_attention_leaves_out_what_a_row_does_not_see(dtype, fresh):
    """Keys and values behind a sequence, of later tokens and before the window are infinite or NaN; pages are missing."""
    import torch
    rng = np.random.default_rng(11)
    heads, kv_heads, d, page, cached, window = 8, 2, 64, 16, [100, 37, 20, 0], 48
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, page, cached, fresh)
    clean = run(q, k, v, table, starts, lengths, max(fresh), window=window)
    check_attention(dtype, q, k, v, table, starts, lengths, clean, d ** -0.5, window)
    bad = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(torch_type(dtype)).min], device="cuda", dtype=torch_type(dtype))
    owned = torch.zeros(k.shape[0] * page, dtype=torch.bool)
    for s, n in enumerate(lengths):
        for j in range(n):
            owned[table[s, j // page] * page + j % page] = True
    for cache in (k, v):
        flat = cache.flatten(0, 1)
        flat[~owned.cuda()] = bad[torch.randint(0, 4, (int((~owned).sum()), kv_heads, d), device="cuda")]
    assert torch.equal(run(q, k, v, table, starts, lengths, max(fresh), window=window), clean)
    # the newest token of the first sequence, and its oldest: only rows that see them change
    for j, sees in ((lengths[0] - 1, [fresh[0] - 1]), (0, [i for i in range(fresh[0]) if cached[0] + i < window])):
        for cache in (k, v):
            flat = cache.flatten(0, 1)
            at, old = table[0, j // page] * page + j % page, None
            old = flat[at].clone()
            flat[at] = bad[:3][torch.randint(0, 3, (kv_heads, d), device="cuda")]
            got = run(q, k, v, table, starts, lengths, max(fresh), window=window)
            flat[at] = old
            blind = [i for i in range(int(starts[-1])) if i not in sees]
            want, size, reach = PO.attention(host(q), host(k), host(v), table, starts, lengths, d ** -0.5, window)
            from paged_util import attention_bound
            off = np.abs(host(got) - want)[blind]
            assert (off <= attention_bound(dtype, want, size, reach, d)[blind]).all()
            if sees:
                assert not torch.isfinite(got[sees]).any(-1).all()
    # pages that do not exist
    table[0, 1], table[1, 2], table[0, 4] = -1, k.shape[0], 2 ** 31 - 1
    k, v = (torch.nan_to_num(x, 0.5, 0.5, 0.5).clamp(-4, 4) for x in (k, v))
    got = run(q, k, v, table, starts, lengths, max(fresh), window=window)
    check_attention(dtype, q, k, v, table, starts, lengths, got, d ** -0.5, window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_rows_that_see_nothing_and_rows_of_nobody(dtype):
    import torch
    rng = np.random.default_rng(2)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, 8, 2, 128, 16, [20, 5, 90], [3, 4, 40], rows=60)
    lengths = np.array([0, 2, 130])                                # the first has no tokens, two rows of the second lie before its start
    before = torch.full_like(q, 3.0)
    got = run(q, k, v, table, starts, lengths, 40, out=before.clone())
    check_attention(dtype, q, k, v, table, starts, lengths, got, 128 ** -0.5, before=host(before))
    assert (got[:5] == 0).all() and (got[47:] == 3.0).all()
    table[2] = -1
    assert (run(q, k, v, table, starts, lengths, 40)[7:47] == 0).all()
    # words out of range are cut off
    got = run(q, k, v, table, [0, 3, 7, 2 ** 31 - 1], [20, 9, 2 ** 31 - 1], 40)
    check_attention(dtype, q, k, v, table, np.array([0, 3, 7, 60]), np.array([20, 9, table.shape[1] * 16]), got, 128 ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_reads_and_writes_rows_any_distance_apart(dtype):
    import torch
    rng = np.random.default_rng(4)
    for pad, d in ((8, 64), (3, 64), (1, 128)):
        q, k, v, table, starts, lengths = attention_inputs(rng, dtype, 4, 2, d, 16, [20, 5], [2, 60])
        wide = torch.full((q.shape[0], 4 * d + pad), 9.0, dtype=q.dtype, device="cuda")
        wide[:, pad:] = q.flatten(1)
        out = torch.full_like(wide, 5.0)
        got = run(wide[:, pad:].unflatten(1, (4, d)), k, v, table, starts, lengths, 60, out=out[:, :4 * d].unflatten(1, (4, d)))
        check_attention(dtype, q, k, v, table, starts, lengths, got, d ** -0.5)
        assert (out[:, 4 * d:] == 5.0).all()


@pytest.mark.parametrize("dtype,fresh", [("bf16", [1, 2]), ("bf16", [60, 3]), ("f32", [2, 1])])
def test_attention_in_a_cache_beyond_32_bit_offsets(dtype, fresh):
    import torch
    heads, kv_heads, d, page, pages = 8, 8, 256 if dtype == "f32" else 128, 64, (1 << 32) // (8 * 128 * 64) + 40
    if dtype == "f32":
        pages = (1 << 32) // (8 * 256 * 64) + 40
    rng = np.random.default_rng(6)
    t = torch_type(dtype)
    total = np.array([130, 200])
    table = np.array([[pages - 1, 3, pages - 7, -1], [pages - 2, 0, pages - 9, pages - 20]])
    k, v = (torch.empty(pages, page, kv_heads, d, dtype=t, device="cuda") for _ in range(2))
    starts = np.concatenate([[0], np.cumsum(fresh)])
    ids = torch.from_numpy(table[table >= 0]).cuda()
    small = []
    for c in (k, v):
        c[ids] = torch.randn(len(ids), page, kv_heads, d, device="cuda").to(t)
        small.append(c[ids])
    local = np.full(table.shape, -1)
    local[table >= 0] = np.arange(len(ids))
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]), heads, d)).astype(np.float32)).cuda().to(t)
    got = run(q, k, v, table, starts, total, max(fresh))
    check_attention(dtype, q, *small, local, starts, total, got, d ** -0.5)
    # and the write into its last rows
    from meganeura_b200 import ops
    x = torch.randn(2, kv_heads, d, device="cuda").to(t)
    ops.paged_append(None, x, x, words([0, 1]), words([pages * page - 1, pages * page - 70]), k, v)
    assert torch.equal(k[-1, -1], x[0]) and torch.equal(v[-2, page - 6], x[1])


def test_attention_of_long_sequences_is_split_and_joined():
    rng = np.random.default_rng(8)
    for dtype, heads, kv_heads, d, cached, fresh in (("bf16", 4, 1, 128, [20000, 3], [1, 1]), ("f16", 8, 2, 64, [9000], [4]), ("f32", 4, 2, 64, [5000], [1]),
                                                     ("bf16", 2, 1, 128, [7000], [100])):
        q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, cached, fresh, gain=2.0)
        check_attention(dtype, q, k, v, table, starts, lengths, run(q, k, v, table, starts, lengths, max(fresh)), d ** -0.5)


@pytest.mark.parametrize("dtype,heads,kv_heads,d,window", [("bf16", 8, 2, 128, 0), ("f16", 6, 3, 64, 0), ("bf16", 8, 2, 80, 700), ("f16", 3, 1, 64, 100),
                                                                 ("f32", 4, 1, 128, 0), ("f32", 3, 3, 52, 300)])
def test_attention_of_long_portions(dtype, heads, kv_heads, d, window):
    """Enough work for several units per CTA and many blocks of keys per unit.  The oracle takes a sample of the rows."""
    rng = np.random.default_rng(17)
    cached, fresh = [3000, 0, 900, 5000], [2100, 2500, 1300, 1000]
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 32, cached, fresh, gain=1.5)
    got = run(q, k, v, table, starts, lengths, 2500, window=window)
    for s in range(4):
        for i in sorted({0, 1, 63, 64, 127, 128, fresh[s] - 1} | set(rng.integers(0, fresh[s], 12).tolist())):
            r, n = int(starts[s]) + i, int(lengths[s]) - fresh[s] + i + 1               # the row alone, as the last token of its sequence
            check_attention(dtype, q[r:r + 1], k, v, table[s:s + 1], [0, 1], [n], got[r:r + 1], d ** -0.5, window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-35])
def test_attention_with_any_scale(dtype, scale):
    rng = np.random.default_rng(21)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, 8, 2, 64, 16, [100, 30], [1, 80])
    check_attention(dtype, q, k, v, table, starts, lengths, run(q, k, v, table, starts, lengths, 80, scale=scale), scale)


@pytest.mark.parametrize("dtype,heads,kv_heads,d", [("bf16", 300, 1, 64), ("f32", 130, 1, 32), ("f16", 256, 2, 128)])
def test_attention_of_very_many_heads_per_key_head(dtype, heads, kv_heads, d):
    rng = np.random.default_rng(22)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 16, [70, 0], [1, 3])
    check_attention(dtype, q, k, v, table, starts, lengths, run(q, k, v, table, starts, lengths, 3), d ** -0.5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 6, 200])
def test_attention_hands_nan_on_to_the_rows_that_see_it(dtype, fresh):
    """NaN in a query makes its row NaN; in a key all heads and rows that see it; neither reaches another row."""
    import torch
    rng = np.random.default_rng(23)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, 4, 2, 128, 16, [90, 50], [fresh, fresh])
    clean = run(q, k, v, table, starts, lengths, fresh)
    q[fresh // 2, 1] = float("nan")
    got = run(q, k, v, table, starts, lengths, fresh)
    assert torch.isnan(got[fresh // 2, 1]).all()
    got[fresh // 2, 1] = clean[fresh // 2, 1]
    assert torch.equal(got, clean)
    q[fresh // 2, 1] = 0.5
    clean = run(q, k, v, table, starts, lengths, fresh)
    k[table[0, 2], 3, 0, 5] = float("nan")
    got = run(q, k, v, table, starts, lengths, fresh)
    assert torch.isnan(got[:fresh, :2]).all()                      # the heads of the first key head
    assert torch.equal(got[:fresh, 2:], clean[:fresh, 2:]) and torch.equal(got[fresh:], clean[fresh:])


def test_attention_with_many_sequences():
    rng = np.random.default_rng(9)
    cached, fresh = rng.integers(0, 40, 4096), rng.integers(0, 3, 4096)
    q, k, v, table, starts, lengths = attention_inputs(rng, "f16", 2, 1, 64, 8, cached, fresh)
    check_attention("f16", q, k, v, table, starts, lengths, run(q, k, v, table, starts, lengths, 2), 0.125)


def test_attention_gives_the_same_bits_again_and_under_any_bound_of_new_tokens_that_holds():
    import torch
    rng = np.random.default_rng(10)
    q, k, v, table, starts, lengths = attention_inputs(rng, "bf16", 16, 4, 128, 16, [900, 40, 0], [4, 200, 33])
    first = run(q, k, v, table, starts, lengths, 200)
    assert all(torch.equal(run(q, k, v, table, starts, lengths, 200), first) for _ in range(3))
    for most in (1, 8, 199, 100000):                               # a bound that does not hold costs time, nothing else
        check_attention("bf16", q, k, v, table, starts, lengths, run(q, k, v, table, starts, lengths, most), 128 ** -0.5)


# ---------------------------------------------------------------------------------------------- probabilities

@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 7, 2), (2, 1000, 0), (5, 4099, 0), (1, 32768, 0), (4, 32768, 4), (70, 5000, 0), (3, 151936, 0), (2, 163841, 3),
                                            (2, 400000, 0), (300, 20484, 0)])
def test_token_probs(rows, vocab, pad):
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(vocab)
    wide = torch.from_numpy((rng.standard_normal((rows, vocab + pad)) * 4).astype(np.float32)).cuda()
    t = (0.2 + rng.random(rows)).astype(np.float32)
    t[rows // 2] = 0.0
    logits = wide[:, :vocab]
    out = torch.full_like(wide, 5.0)
    got = ops.token_probs(logits, torch.from_numpy(t).cuda(), out=out[:, :vocab])
    want = PO.probs(host(logits), t)
    # the exponent (x - m) / t is off by 2^-22 of its size, which is at most 104 where a weight is not below f32's range; the exponential 2^-22, the sum 2^-18
    spread = np.minimum(104.0, (host(logits).max(1, keepdims=True) - host(logits)) / np.maximum(t, 1e-30)[:, None])
    # below f32's normal range a weight is a multiple of 2^-149: expf's two units in the last place are 2 * 2^-149 there, the product with 1 / sum <= 1
    # keeps that at most and rounds by half a unit more
    off, bound = np.abs(host(got) - want), want * (2.0 ** -22 * (spread + 1) + 2.0 ** -18) + 2.5 * 2.0 ** -149
    at = np.unravel_index((off - bound).argmax(), off.shape)
    assert off[at] <= bound[at], (at, host(got)[at], want[at])
    assert (out[:, vocab:] == 5.0).all()
    assert torch.equal(ops.token_probs(logits), ops.token_probs(logits, torch.ones(rows, device="cuda")))


@pytest.mark.parametrize("dtype,heads,kv_heads,d,fresh", [
    ("f32", 1, 1, 64, 1), ("f32", 4, 1, 128, 1), ("f32", 7, 1, 64, 1), ("f32", 4, 2, 80, 7), ("f32", 8, 1, 128, 3), ("f32", 2, 1, 64, 40), ("f32", 2, 1, 256, 1),
    ("bf16", 4, 1, 128, 1), ("f16", 4, 1, 64, 5), ("bf16", 4, 1, 128, 60),
])
@pytest.mark.parametrize("slope", [1 / 64, 1.0, -1.0, 40.0])
def test_attention_whose_scores_rise_or_fall_from_key_to_key(dtype, heads, kv_heads, d, fresh, slope):
    import torch
    rng = np.random.default_rng(d + fresh)
    q, k, v, table, starts, lengths = attention_inputs(rng, dtype, heads, kv_heads, d, 16, [333, 90], [fresh, fresh])
    q[..., 0], q[..., 1:] = 4.0, q[..., 1:] / 64                   # scores: slope * position, and a little of the rest
    flat = k.flatten(0, 1)
    for s, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        flat[torch.from_numpy(table[s]).cuda()[at // 16] * 16 + at % 16, :, 0] = (slope / 4 * at.float()).to(k.dtype)[:, None]
    check_attention(dtype, q, k, v, table, starts, lengths, run(q, k, v, table, starts, lengths, fresh, scale=1.0), 1.0)


def test_token_probs_in_place():
    import torch
    from meganeura_b200 import ops
    for rows, vocab in ((3, 999), (2, 5000), (5, 40000)):
        x = torch.randn(rows, vocab, device="cuda")
        want = ops.token_probs(x)
        assert torch.equal(ops.token_probs(x, out=x), want) and x.data_ptr() == ops.token_probs(x, out=x).data_ptr()


def test_token_probs_of_rows_with_infinities_nan_and_ties():
    import torch
    from meganeura_b200 import ops
    inf, nan = math.inf, math.nan
    rows = np.array([[1, 2, 2, nan], [-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [inf, 1, inf, 0], [-inf, 3, nan, -inf], [0, 0, 0, 0], [-3e38, 3e38, 0, 1]], np.float32)
    for t in (1.0, 0.0, 1e-40, -1.0, nan):
        temp = np.full(len(rows), t, np.float32)
        got = host(ops.token_probs(torch.from_numpy(rows).cuda(), torch.from_numpy(temp).cuda()))
        assert np.allclose(got, PO.probs(rows, temp), rtol=1e-6, atol=1e-30), t


# ---------------------------------------------------------------------------------------------- verification of drafts

def verify_case(rng, sequences, most, vocab, sampled, sharp=3.0):
    import torch
    n = rng.integers(0, most + 2, sequences)
    n[0] = max(n[0], 1)
    starts = np.concatenate([[0], np.cumsum(n)])
    rows = int(starts[-1])
    logits = rng.standard_normal((rows, vocab)) * sharp
    soft = lambda x: (np.exp(x - x.max(1, keepdims=True)) / np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)).astype(np.float32)  # noqa: E731
    p, q = soft(logits), soft(logits + 0.7 * rng.standard_normal((rows, vocab)))
    tokens = np.roll(np.array([rng.choice(vocab, p=row.astype(np.float64) / row.sum(dtype=np.float64)) for row in (q if sampled else p)]), 1)
    return p, (q if sampled else None), tokens, starts, rng.random(rows).astype(np.float32), rng.random(sequences).astype(np.float32), torch


def check_verify(p, q, tokens, starts, accept, sample, torch):
    from meganeura_b200 import ops
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    out = tuple(torch.full((n,), -2, dtype=torch.int32, device="cuda") for n in (len(sample), len(sample), len(tokens)))
    got = ops.verify_drafts(dev(p), None if q is None else dev(q), words(tokens), words(starts), dev(accept), dev(sample), out=out)
    for name, have, want in zip(("accepted", "next", "out"), got, PO.verify(p, q, tokens, starts, accept, sample)):
        assert np.array_equal(host(have), want), name
    return got


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("sequences,most,vocab", [(1, 0, 1), (1, 3, 5), (4, 4, 1001), (3, 8, 32768), (40, 2, 2052), (2, 3, 151936), (2, 2, 170001), (700, 1, 64), (1, 1200, 33)])
def test_verify_drafts(sampled, sequences, most, vocab):
    rng = np.random.default_rng(vocab + most)
    check_verify(*verify_case(rng, sequences, most, vocab, sampled))


def test_verify_drafts_at_the_borders():
    rng = np.random.default_rng(1)
    p, q, tokens, starts, accept, sample, torch = verify_case(rng, 6, 3, 3000, True)
    for u in (0.0, 1.0, math.nan, -1.0, 2.0, 1 - 2.0 ** -24):
        check_verify(p, q, tokens, starts, np.full_like(accept, 0.9), np.full_like(sample, u), torch)
        check_verify(p, q, tokens, starts, np.full_like(accept, u), sample, torch)
    check_verify(p, p, tokens, starts, np.ones_like(accept), sample, torch)                    # refused at u = 1 with nothing left over: from p itself
    check_verify(p, None, tokens, starts, np.ones_like(accept), sample, torch)
    check_verify(p, q, np.full_like(tokens, -1), starts, accept, sample, torch)                # no drafts after all
    check_verify(p, q, np.full_like(tokens, 3000), starts, accept, sample, torch)
    check_verify(np.zeros_like(p), q, tokens, starts, accept, sample, torch)                   # no mass anywhere
    holes = p.copy()
    holes[:, ::3], holes[:, 1::5], holes[:, 2::7] = np.nan, np.inf, -1.0
    check_verify(holes, q, tokens, starts, accept, sample, torch)
    check_verify(p, holes, tokens, starts, accept, sample, torch)
    one = np.zeros_like(p)
    one[np.arange(len(p)), rng.integers(0, 3000, len(p))] = 1
    check_verify(one, None, tokens, starts, accept, sample, torch)
    check_verify(p, q, tokens, np.minimum(starts, starts[-1] - 2), accept, sample, torch)      # rows behind the last sequence stay
    over = starts.copy()
    over[-1] += 1000
    check_verify(p, q, tokens, over, accept, sample, torch)


# ---------------------------------------------------------------------------------------------- together

class Server:
    """Chats over one cache: what a program that serves them keeps, and a step as it runs it."""

    def __init__(self, torch, ops, sequences, rows, heads, kv_heads, d, vocab, page, pages, dtype, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        t = torch_type(dtype)
        self.shape, self.ops, self.torch = (heads, kv_heads, d), ops, torch
        self.embed = torch.randn(vocab, (heads + 2 * kv_heads) * d, device="cuda", generator=g)
        self.head = torch.randn(heads * d, vocab, device="cuda", generator=g) * 0.3
        self.k, self.v = (torch.full((pages, page, kv_heads, d), float("nan"), device="cuda").to(t) for _ in range(2))
        self.page, self.rows = page, rows
        self.table = torch.full((sequences, pages), -1, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(sequences, dtype=torch.int32, device="cuda")
        self.free, self.count = torch.randperm(pages, device="cuda", generator=g).int(), words([pages])
        self.step_ = ops.PagedStep.empty(sequences, rows)
        self.logits = None

    def forward(self, tokens, cached, fresh, most):
        """The model: a step's logits."""
        o, (h, kv, d) = self.ops, self.shape
        o.paged_plan(cached, fresh, self.table, self.held, self.free, self.count, self.page, self.rows, step=self.step_)
        s = self.step_
        q, k, v = (x.unflatten(1, (-1, d)) for x in self.embed[tokens.long().clamp(min=0)].split([h * d, kv * d, kv * d], 1))
        q = o.paged_append(q, k, v, s.positions, s.slots, self.k, self.v, theta=1e4)
        x = o.paged_attention(q, self.k, self.v, self.table, s.starts, s.lengths, most)
        return x.flatten(1).float() @ self.head

    def trim(self, lengths):
        self.ops.paged_trim(lengths, self.table, self.held, self.free, self.count, self.page)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_serving_loop_agrees_with_its_restatement_token_by_token(dtype):
    """Prompts in portions, then drafted tokens, verified, the rejected ones taken back, a chat that ends and gives its pages to the others.  The
    restatement keeps each chat's tokens in a list and computes its logits from scratch; the operators' probabilities go into its verification."""
    import torch
    from meganeura_b200 import ops
    heads, kv_heads, d, vocab, page, pages, rows, n = 4, 2, 64, 97, 8, 60, 64, 3
    sv = Server(torch, ops, n, rows, heads, kv_heads, d, vocab, page, pages, dtype, 5)
    rng = np.random.default_rng(12)
    chats = [list(rng.integers(0, vocab, m)) for m in (50, 7, 90)]
    cached = np.zeros(n, np.int64)
    embed, head = host(sv.embed).astype(np.float64), host(sv.head).astype(np.float64)
    cut = lambda x: x.to(torch_type(dtype)).double().cpu().numpy()  # noqa: E731

    def plain(chat):
        """Logits behind every token of a chat."""
        x = embed[chat]
        pos = np.arange(len(chat))
        q, k, v = (y.reshape(len(chat), -1, d) for y in np.split(x, [heads * d, (heads + kv_heads) * d], 1))
        q, k, v = (cut(torch.from_numpy(y)) for y in (PO.rotate(q, pos, 1e4), PO.rotate(k, pos, 1e4), v))
        pages_ = np.arange(-(-len(chat) // 8))[None]
        pad = lambda y: np.concatenate([y, np.zeros((pages_.size * 8 - len(chat),) + y.shape[1:])]).reshape(-1, 8, kv_heads, d)  # noqa: E731
        o = PO.attention(q, pad(k), pad(v), pages_, [0, len(chat)], [len(chat)], d ** -0.5)[0]
        return o.reshape(len(chat), -1) @ head

    def close(got, want):
        assert np.abs(got - want).max() <= (1e-3 if dtype == "f32" else 0.15) * np.abs(want).max()

    def step(fed):
        """Feeds lists of tokens; the logits of each."""
        flat = [t for f in fed for t in f]
        fresh = np.array([len(f) for f in fed])
        logits = sv.forward(words(flat + [-1] * (rows - len(flat))), words(cached), words(fresh), int(fresh.max()))
        assert int(host(sv.step_.lacking)[0]) == 0
        return logits

    done = np.zeros(n, np.int64)
    while any(done[i] < len(chats[i]) - 1 for i in range(n)):                       # prompts, 20 tokens at a time, the last token kept back
        fed = [chats[i][done[i]:min(done[i] + 20, len(chats[i]) - 1)] for i in range(n)]
        logits = host(step(fed))
        at = 0
        for i, f in enumerate(fed):
            if f:
                close(logits[at:at + len(f)], plain(chats[i][:done[i] + len(f)])[done[i]:])
            at += len(f)
            done[i] += len(f)
        cached = done.copy()
    for turn in range(8):
        live = [i for i in range(n) if not (turn >= 4 and i == 1)]
        if turn == 4:                                                               # the second chat ends
            cached[1] = 0
            sv.trim(words(cached))
        drafts = [list(rng.integers(0, vocab, rng.integers(0, 4))) if i in live else [] for i in range(n)]
        fed = [[chats[i][-1]] + drafts[i] if i in live else [] for i in range(n)]
        logits = step(fed)
        p = ops.token_probs(logits[:sum(map(len, fed))].contiguous())
        total, flat, starts = p.shape[0], [t for f in fed for t in f], np.concatenate([[0], np.cumsum([len(f) for f in fed])])
        q = torch.full_like(p, 1 / vocab)
        accept, sample = rng.random(total).astype(np.float32) * 0.2, rng.random(n).astype(np.float32)
        got = ops.verify_drafts(p, q, words(flat), words(starts), torch.from_numpy(accept).cuda(), torch.from_numpy(sample).cuda())
        want = PO.verify(host(p), host(q), np.array(flat), starts, accept, sample)
        for a, b in zip(got, want):
            assert np.array_equal(host(a)[:len(b)], b)
        for i in live:
            full = plain(chats[i] + drafts[i])
            close(host(logits)[starts[i]:starts[i + 1]], full[len(chats[i]) - 1:])
            kept = int(want[0][i])
            cached[i] = len(chats[i]) + kept
            chats[i] += drafts[i][:kept] + [int(want[1][i])]
        sv.trim(words(cached))
        assert int(host(sv.count)[0]) == pages - sum(-(-int(c) // page) for c in cached)


def test_a_captured_step_replays_with_other_lengths_beside_another_graph():
    """One graph per layout of a step; lengths, tokens and pages change between replays.  Two graphs of the same cache replay on two streams."""
    import torch
    from meganeura_b200 import ops
    sv = Server(torch, ops, 3, 12, 8, 2, 64, 50, 16, 40, "bf16", 3)
    tokens, cached, fresh = words(np.zeros(12)), words([0, 0, 0]), words([1, 1, 1])
    sv.forward(tokens, cached, fresh, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = sv.forward(tokens, cached, fresh, 4)
        probs = ops.token_probs(logits)
        picked = ops.verify_drafts(probs, None, tokens, sv.step_.starts, torch.full((12,), 0.5, device="cuda"), torch.full((3,), 0.5, device="cuda"))
    rng = np.random.default_rng(3)
    have = np.zeros(3, np.int64)
    eager = Server(torch, ops, 3, 12, 8, 2, 64, 50, 16, 40, "bf16", 3)
    for turn in range(6):
        n = rng.integers(0, 5, 3)
        tok = rng.integers(0, 50, 12)
        tokens.copy_(words(tok)), cached.copy_(words(have)), fresh.copy_(words(n))
        graph.replay()
        want = eager.forward(words(tok), words(have), words(n), 4)
        total = int(n.sum())
        assert torch.equal(logits[:total], want[:total])
        assert torch.equal(probs[:total], ops.token_probs(want)[:total])
        have += n
    q, k, v, table, starts, lengths = attention_inputs(rng, "bf16", 8, 2, 128, 16, [3000, 700], [1, 1])
    q2 = q.flip(0).contiguous()
    args = (words(table), words(starts), words(lengths), 1)
    alone = [ops.paged_attention(x, k, v, *args) for x in (q, q2)]
    graphs, outs = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention(x, k, v, *args))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for have_, want in zip(outs, alone):
        assert torch.equal(have_, want)


def test_calls_on_a_stream_of_their_own():
    import torch
    from meganeura_b200 import ops
    rng = np.random.default_rng(13)
    q, k, v, table, starts, lengths = attention_inputs(rng, "f16", 8, 2, 64, 16, [500, 3], [2, 70])
    args = (words(table), words(starts), words(lengths), 70)
    want = ops.paged_attention(q, k, v, *args)
    probs = ops.token_probs(q.flatten(1).float())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got, p = ops.paged_attention(q, k, v, *args, stream=side), ops.token_probs(q.flatten(1).float(), stream=side)
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(p, probs)


def test_python_checks_name_what_is_wrong():
    import torch
    from meganeura_b200 import MgqError, ops
    rng = np.random.default_rng(14)
    q, k, v, table, starts, lengths = attention_inputs(rng, "f16", 8, 2, 64, 16, [5], [1])
    t, s, n = words(table), words(starts), words(lengths)
    for bad in (lambda: ops.paged_attention(q.float(), k, v, t, s, n, 1), lambda: ops.paged_attention(q, k, v[..., :32], t, s, n, 1),
                lambda: ops.paged_attention(q, k, v, t.long(), s, n, 1), lambda: ops.paged_attention(q, k, v, t, s[:1], n, 1), lambda: ops.paged_attention(q, k, v, t, s, n, 1, window=-1),
                lambda: ops.paged_attention(q.expand(3, -1, -1), k, v, t, s, n, 1), lambda: ops.paged_attention(q.transpose(1, 2), k, v, t, s, n, 1),
                lambda: ops.paged_append(q, q[:, :2], q[:, :2], s[:1], s[:1], k.float(), v.float()), lambda: ops.paged_append(q, q[:, :3], q[:, :3], s[:1], s[:1], k, v),
                lambda: ops.paged_plan(s, n, t, n, n, n, 16, 4), lambda: ops.token_probs(q[:, 0]), lambda: ops.token_probs(q[:, 0].float(), torch.ones(3, device="cuda")),
                lambda: ops.verify_drafts(q[:, 0].float(), q[:, 0], n, s, q[0, 0, :1].float(), q[0, 0, :1].float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(MgqError) as e:
        ops.paged_attention(q[:, :7].contiguous(), k, v, t, s, n, 1)
    assert e.value.status == 2
    with pytest.raises(MgqError):
        ops.paged_plan(n, n, t, n, n, n, 12, 1)
