"""The 8-bit operators at the ends of what their documentation allows."""
import numpy as np
import pytest

from int8_util import attention_inputs, check_attention

pytestmark = pytest.mark.gpu


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


def test_no_wait_ran_out():
    from meganeura_b200 import ops
    ops.device_status()
