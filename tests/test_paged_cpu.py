"""Argument checks of the operators over a paged cache, and the oracle's own invariants: no GPU needed."""
import numpy as np
import pytest

from meganeura_b200 import _lib
from oracle import paged_oracle as PO

OK, NULL, SHAPE, FORMAT, ALIGN = 0, 1, 2, 3, 7
P = 4096                     # a pointer that no call follows: every call below is refused before it touches the device


def plan(**change):
    a = dict(cached=P, fresh=P, sequences=4, page_size=16, table=P, width=8, held=P, free=P, pages=32, count=P, rows=16, starts=P, lengths=P, positions=P, slots=P, lacking=P)
    a.update(change)
    return _lib.lib.mgq_paged_plan(*a.values(), None)


def trim(**change):
    a = dict(lengths=P, sequences=4, page_size=16, table=P, width=8, held=P, free=P, pages=32, count=P)
    a.update(change)
    return _lib.lib.mgq_paged_trim(*a.values(), None)


def append(**change):
    a = dict(q=P, k=P, v=P, src=0, positions=P, slots=P, q_out=P, k_cache=P, v_cache=P, dtype=0, rows=4, heads=8, kv_heads=2, d=64, q_pitch=512, k_pitch=128, v_pitch=128,
             page_size=16, pages=32, theta=1e4)
    a.update(change)
    return _lib.lib.mgq_paged_append(*a.values(), None)


def attention(**change):
    a = dict(q=P, k=P, v=P, dtype=1, table=P, starts=P, lengths=P, out=P, sequences=2, rows=4, max_fresh=2, heads=8, kv_heads=2, d=64, page_size=16, pages=32, width=8,
             q_pitch=512, out_pitch=512, scale=0.125, window=0, workspace=P)
    a.update(change)
    return _lib.lib.mgq_paged_attention(*a.values(), None)


def probs(**change):
    a = dict(logits=P, pitch=100, temperature=None, out=P, out_pitch=100, rows=3, vocab=100)
    a.update(change)
    return _lib.lib.mgq_token_probs(*a.values(), None)


def verify(**change):
    a = dict(target=P, t_pitch=100, draft=P, d_pitch=100, tokens=P, starts=P, accept=P, sample=P, accepted=P, next=P, out=P, sequences=2, rows=6, vocab=100)
    a.update(change)
    return _lib.lib.mgq_verify_drafts(*a.values(), None)


def test_append_in_place_needs_dense_queries_of_the_caches_type():
    assert append(q_pitch=600) == SHAPE and append(dtype=1) == SHAPE and append(src=0, dtype=4) == SHAPE


@pytest.mark.parametrize("call,change,status", [
    *[(plan, {name: None}, NULL) for name in ("cached", "fresh", "table", "held", "free", "count", "starts", "lengths", "positions", "slots", "lacking")],
    (plan, dict(page_size=12), SHAPE), (plan, dict(page_size=4), SHAPE), (plan, dict(page_size=2048), SHAPE), (plan, dict(pages=0), SHAPE),
    (plan, dict(pages=1 << 28), SHAPE), (plan, dict(sequences=0), SHAPE), (plan, dict(sequences=4097), SHAPE), (plan, dict(width=0), SHAPE),
    (plan, dict(width=1 << 26), SHAPE), (plan, dict(rows=0), SHAPE), (plan, dict(rows=1 << 31), SHAPE),
    *[(trim, {name: None}, NULL) for name in ("lengths", "table", "held", "free", "count")],
    (trim, dict(page_size=24), SHAPE), (trim, dict(sequences=5000), SHAPE), (trim, dict(width=0), SHAPE),
    *[(append, {name: None}, NULL) for name in ("k", "v", "positions", "slots", "k_cache", "v_cache", "q_out")],
    (append, dict(dtype=2), FORMAT), (append, dict(src=1, dtype=4), FORMAT), (append, dict(src=4, dtype=0), FORMAT), (append, dict(heads=9), SHAPE),
    (append, dict(heads=0), SHAPE), (append, dict(kv_heads=0), SHAPE), (append, dict(d=63), SHAPE), (append, dict(d=258), SHAPE), (append, dict(d=0), SHAPE),
    (append, dict(rows=0), SHAPE), (append, dict(q_pitch=511), SHAPE), (append, dict(k_pitch=127), SHAPE), (append, dict(v_pitch=0), SHAPE),
    (append, dict(theta=-1.0), SHAPE), (append, dict(theta=float("nan")), SHAPE), (append, dict(theta=float("inf")), SHAPE), (append, dict(page_size=7), SHAPE),
    (append, dict(k=P + 2), ALIGN), (append, dict(dtype=1, k_cache=P + 1), ALIGN),
    *[(attention, {name: None}, NULL) for name in ("q", "k", "v", "table", "starts", "lengths", "out", "workspace")],
    (attention, dict(dtype=3), FORMAT), (attention, dict(heads=7), SHAPE), (attention, dict(heads=0), SHAPE), (attention, dict(kv_heads=0), SHAPE),
    (attention, dict(d=257, q_pitch=4096, out_pitch=4096), SHAPE), (attention, dict(d=0), SHAPE), (attention, dict(rows=0), SHAPE), (attention, dict(max_fresh=0), SHAPE),
    (attention, dict(q_pitch=500), SHAPE), (attention, dict(out_pitch=500), SHAPE), (attention, dict(sequences=0), SHAPE), (attention, dict(width=0), SHAPE),
    (attention, dict(pages=0), SHAPE), (attention, dict(page_size=33), SHAPE), (attention, dict(q=P + 1), ALIGN), (attention, dict(dtype=0, out=P + 2), ALIGN),
    (attention, dict(workspace=P + 8), ALIGN),
    (probs, dict(logits=None), NULL), (probs, dict(out=None), NULL), (probs, dict(rows=0), SHAPE), (probs, dict(vocab=0), SHAPE), (probs, dict(pitch=99), SHAPE),
    (probs, dict(out_pitch=99), SHAPE),
    *[(verify, {name: None}, NULL) for name in ("target", "tokens", "starts", "accept", "sample", "accepted", "next", "out")],
    (verify, dict(sequences=0), SHAPE), (verify, dict(rows=0), SHAPE), (verify, dict(vocab=0), SHAPE), (verify, dict(t_pitch=99), SHAPE), (verify, dict(d_pitch=99), SHAPE),
])
def test_refusals(call, change, status):
    assert call(**change) == status
    assert _lib.last_error()


def test_workspace_of_arguments_that_are_refused_is_zero():
    size = _lib.lib.mgq_paged_attention_workspace
    assert size(8, 2, 64, 1, 1) > 0 and size(32, 8, 128, 2048, 4) > 0
    assert size(8, 3, 64, 1, 1) == size(8, 0, 64, 1, 1) == size(8, 2, 300, 1, 1) == size(8, 2, 64, 0, 1) == size(8, 2, 64, 1, 2) == size(0, 2, 64, 1, 1) == 0


def test_host_tensors_are_refused():
    import torch
    from meganeura_b200 import ops
    w = torch.zeros(4, dtype=torch.int32)
    cache = torch.zeros(2, 16, 2, 64)
    with pytest.raises(ValueError):
        ops.paged_plan(w, w, torch.zeros(4, 2, dtype=torch.int32), w, w, w[:1], 16, 8)
    with pytest.raises(ValueError):
        ops.paged_trim(w, torch.zeros(4, 2, dtype=torch.int32), w, w, w[:1], 16)
    with pytest.raises(ValueError):
        ops.paged_append(None, cache[0], cache[0], w, w, cache, cache)
    with pytest.raises(ValueError):
        ops.paged_attention(cache[0], cache, cache, w[None], w, w, 1)
    with pytest.raises(ValueError):
        ops.token_probs(torch.zeros(2, 8))
    with pytest.raises(ValueError):
        ops.verify_drafts(torch.zeros(2, 8), None, w, w, w, w)


def test_a_trim_to_the_lengths_before_a_plan_undoes_it():
    rng = np.random.default_rng(3)
    for _ in range(50):
        s, page, pages = int(rng.integers(1, 9)), 8, 40
        cached = rng.integers(0, 30, s)
        order, held, table, used = rng.permutation(pages), -(-cached // page), np.full((s, 9), -1), 0
        for i in range(s):
            table[i, :held[i]] = order[used:used + held[i]]
            used += held[i]
        if used > pages:
            continue
        free = np.full(pages, -1)
        free[:pages - used] = order[used:]
        out = PO.plan(cached, rng.integers(0, 40, s), table, held, free, pages - used, page, 60)
        back = PO.trim(cached, out[5], out[6], free, out[7], page)
        for have, want in zip(back, (table, held, free, pages - used)):
            assert np.array_equal(have, want)
