"""Refusals of the operators over a paged cache that need no GPU, beyond those of shapes and types."""
import pytest

from test_paged_cpu import ALIGN, P, append, attention, plan, probs, trim, verify


@pytest.mark.parametrize("call,names", [
    (plan, "cached fresh table held free count starts lengths positions slots lacking"), (trim, "lengths table held free count"), (append, "positions slots"),
    (attention, "table starts lengths"), (probs, "logits temperature out"), (verify, "target draft tokens starts accept sample accepted next out"),
])
def test_words_and_floats_at_odd_addresses_are_refused(call, names):
    for name in names.split():
        for off in (1, 2, 3):
            assert call(**{name: P + off}) == ALIGN, name
