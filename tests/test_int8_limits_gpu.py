"""The 8-bit operators at the ends of what their documentation allows."""
import numpy as np
import pytest

from int8_util import attention_bound, attention_inputs, check_attention
from oracle import int8_oracle as IO
from oracle import paged_oracle as PO
from paged_util import host, words

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


def test_no_wait_ran_out():
    from meganeura_b200 import ops
    ops.device_status()
