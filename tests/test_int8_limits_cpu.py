"""What the operators of 8-bit integers refuse beyond single arguments, without a GPU."""
import pytest

from meganeura_b200 import _lib
from test_int8_cpu import SHAPE, matmul


@pytest.mark.parametrize("change", [dict(out_pitch=101), dict(addend_pitch=128), dict(addend_pitch=104, out_pitch=112, m=2), dict(dtype=0, out_pitch=300, m=300)])
def test_an_addend_in_place_has_the_pitch_of_the_result(change):
    """Else elements would be written before another thread has read them as an addend."""
    assert matmul(**change) == SHAPE
    assert "addend" in _lib.last_error()
