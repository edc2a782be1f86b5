"""The operators of 8-bit integers without a GPU: their restatement, and every argument that is refused."""
import numpy as np
import pytest

from meganeura_b200 import _lib
from oracle import int8_oracle as IO

NULL, SHAPE, FORMAT, ALIGN = 1, 2, 3, 7
P = 1 << 20                                              # an address that is never followed


def quantize(**change):
    a = dict(x=P, dtype=4, pitch=96, codes=P, scales=P, rows=4, k=96) | change
    return _lib.lib.mgq_quantize_rows(a["x"], a["dtype"], a["pitch"], a["codes"], a["scales"], a["rows"], a["k"], None)


def matmul(**change):
    a = dict(a=P, a_scales=P, w=P, w_scales=P, addend=P, out=P, dtype=4, m=4, k=64, n=100, addend_pitch=100, out_pitch=100) | change
    return _lib.lib.mgq_matmul_int8(*a.values(), None)


def append(**change):
    a = dict(q=P, k=P, v=P, src=0, positions=P, slots=P, q_out=P, dtype=4, k_cache=P, v_cache=P, k_scales=P, v_scales=P, rows=4, heads=8, kv_heads=2, d=64, q_pitch=512,
             k_pitch=128, v_pitch=128, page_size=32, pages=10, block=16, theta=1e4) | change
    return _lib.lib.mgq_paged_append_int8(*a.values(), None)


def attention(**change):
    a = dict(q=P, k=P, v=P, k_scales=P, v_scales=P, dtype=4, table=P, starts=P, lengths=P, out=P, sequences=3, rows=4, max_fresh=2, heads=8, kv_heads=2, d=64, page_size=32,
             pages=10, block=16, width=4, q_pitch=512, out_pitch=512, scale=0.125, window=0, workspace=P) | change
    return _lib.lib.mgq_paged_attention_int8(*a.values(), None)


@pytest.mark.parametrize("call,change,status", [
    *[(quantize, {name: None}, NULL) for name in ("x", "codes", "scales")],
    (quantize, dict(dtype=2), FORMAT), (quantize, dict(rows=0), SHAPE), (quantize, dict(k=0), SHAPE), (quantize, dict(pitch=95), SHAPE), (quantize, dict(rows=1 << 31), SHAPE),
    (quantize, dict(x=P + 1), ALIGN), (quantize, dict(dtype=0, x=P + 2), ALIGN), (quantize, dict(scales=P + 2), ALIGN),
    *[(matmul, {name: None}, NULL) for name in ("a", "a_scales", "w", "w_scales", "out")],
    (matmul, dict(dtype=3), FORMAT), (matmul, dict(m=0), SHAPE), (matmul, dict(n=0), SHAPE), (matmul, dict(k=0), SHAPE), (matmul, dict(k=72), SHAPE),
    (matmul, dict(k=131072), SHAPE), (matmul, dict(out_pitch=99), SHAPE), (matmul, dict(addend_pitch=99), SHAPE), (matmul, dict(a=P + 8), ALIGN), (matmul, dict(w=P + 4), ALIGN),
    (matmul, dict(out=P + 1), ALIGN), (matmul, dict(dtype=0, addend=P + 2), ALIGN), (matmul, dict(w_scales=P + 1), ALIGN),
    *[(append, {name: None}, NULL) for name in ("k", "v", "positions", "slots", "k_cache", "v_cache", "k_scales", "v_scales", "q_out")],
    (append, dict(dtype=0), FORMAT), (append, dict(src=1, dtype=4), FORMAT), (append, dict(src=3), FORMAT), (append, dict(heads=9), SHAPE), (append, dict(heads=0), SHAPE),
    (append, dict(kv_heads=0), SHAPE), (append, dict(d=72), SHAPE), (append, dict(d=272, q_pitch=4096, k_pitch=4096, v_pitch=4096), SHAPE), (append, dict(rows=0), SHAPE),
    (append, dict(q_pitch=511), SHAPE), (append, dict(k_pitch=127), SHAPE), (append, dict(v_pitch=0), SHAPE), (append, dict(theta=-1.0), SHAPE),
    (append, dict(theta=float("nan")), SHAPE), (append, dict(page_size=48), SHAPE), (append, dict(block=8), SHAPE), (append, dict(block=64), SHAPE), (append, dict(block=24), SHAPE),
    (append, dict(page_size=8, block=8), SHAPE), (append, dict(pages=1 << 27), SHAPE), (append, dict(k_cache=P + 8), ALIGN), (append, dict(k=P + 2), ALIGN),
    (append, dict(v_scales=P + 2), ALIGN), (append, dict(q_out=P), SHAPE),
    *[(attention, {name: None}, NULL) for name in ("q", "k", "v", "k_scales", "v_scales", "table", "starts", "lengths", "out", "workspace")],
    (attention, dict(dtype=0), FORMAT), (attention, dict(heads=7), SHAPE), (attention, dict(heads=0), SHAPE), (attention, dict(d=40), SHAPE), (attention, dict(rows=0), SHAPE),
    (attention, dict(max_fresh=0), SHAPE), (attention, dict(q_pitch=500), SHAPE), (attention, dict(out_pitch=500), SHAPE), (attention, dict(sequences=0), SHAPE),
    (attention, dict(width=0), SHAPE), (attention, dict(pages=0), SHAPE), (attention, dict(block=64), SHAPE), (attention, dict(block=0), SHAPE), (attention, dict(q=P + 1), ALIGN),
    (attention, dict(v=P + 8), ALIGN), (attention, dict(workspace=P + 8), ALIGN), (attention, dict(k_scales=P + 1), ALIGN),
])
def test_refusals(call, change, status):
    if call is append and change == dict(q_out=P):
        change = dict(q_out=P, src=0, q=P)               # in place, but of another type
    assert call(**change) == status
    assert _lib.last_error()


def test_workspace_of_arguments_that_are_refused_is_zero():
    size = _lib.lib.mgq_paged_attention_int8_workspace
    assert size(8, 2, 64, 1) > 0 and size(32, 8, 128, 2048) > 0 and size(8, 1, 256, 5) > 0
    assert size(8, 3, 64, 1) == size(8, 0, 64, 1) == size(8, 2, 272, 1) == size(8, 2, 72, 1) == size(8, 2, 64, 0) == size(0, 2, 64, 1) == 0


def test_host_tensors_are_refused():
    import torch
    from meganeura_b200 import ops
    w, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    codes, cache, scales = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(2, 1, 2)
    with pytest.raises(ValueError):
        ops.quantize_rows(torch.zeros(4, 64))
    with pytest.raises(ValueError):
        ops.matmul_int8(codes, f, codes, f)
    with pytest.raises(ValueError):
        ops.paged_append_int8(None, f, f, w, w, cache, cache, scales, scales)
    with pytest.raises(ValueError):
        ops.paged_attention_int8(cache[0].half(), cache, cache, scales, scales, w[None], w, w, 1)


def test_rows_come_back_within_half_a_code():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((9, 333)) * np.exp2(rng.integers(-90, 100, (9, 1)))).astype(np.float32)
    x[3] = 0
    codes, scales = IO.quantize_rows(x)
    # half a code, and the roundings of 1/127 (half as much), scale, inverse and product: 3.5 * 2^-24 of up to 127 codes
    assert (np.abs(codes * scales[:, None].astype(np.float64) - x) <= scales[:, None] * (0.5 + 127 * 4 * 2.0 ** -24)).all()
    assert (np.abs(codes).max(1) == np.where(scales > 0, 127, 0)).all() and scales[3] == 0


def test_values_that_are_not_finite():
    x = np.ones((4, 16), np.float32)
    x[1, 3], x[2, 5], x[3] = np.nan, -np.inf, 1e-31
    codes, scales = IO.quantize_rows(x)
    assert scales[0] == np.float32(1 / 127) and np.isnan(scales[1]) and scales[2] == np.inf and scales[3] == 0
    assert (codes[1:] == 0).all() and (codes[0] == 127).all()


def test_a_block_keeps_what_it_holds_until_its_first_slot_is_written():
    rng = np.random.default_rng(1)
    cache, scales = np.zeros((3, 32, 2, 16), np.int8), np.full((3, 2, 2), np.nan, np.float32)
    x = rng.standard_normal((40, 2, 16)).astype(np.float32)
    x[20] *= 50
    for r in range(20):                                  # token by token into blocks 2 and 3: slots 32 to 51
        cache, scales = IO.append(cache, scales, x[r:r + 1], [32 + r])
    before = IO.values(cache, scales)[1, :20]
    assert (np.abs(before - x[:20]) <= np.repeat(scales[1], 16, 0)[:20, :, None] * 1.01).all()           # a rounding when written, one or a few when the scale grew
    cache, scales = IO.append(cache, scales, x[20:21], [52])                                           # far larger: the block's older codes are rounded again
    after = IO.values(cache, scales)[1]
    assert np.array_equal(after[:16], before[:16]) and (np.abs(after[16:20] - before[16:20]) <= 0.5001 * scales[1, 1][None, :, None]).all()
    assert (np.abs(after[20] - x[20]) <= 0.5001 * scales[1, 1][:, None]).all()
    cache, scales = IO.append(cache, scales, x[0:3], [48, 49, -1])                                     # anew
    assert (scales[1, 1] < 0.1).all() and np.isnan(scales[0]).all()
