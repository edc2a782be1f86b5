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


def child(code):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]


def test_all_of_ops_is_imported_without_torch_and_its_lazy_names_are_found():
    child("import sys; sys.modules['torch'] = None\n"
          "from meganeura_b200.ops import *\n"
          "from meganeura_b200 import ops\n"
          "assert callable(matmul) and 'paged_plan' in dir(ops)\n")
    child("from meganeura_b200 import ops\nassert callable(ops.verify_drafts) and ops.NO_SLOT == -1\n")


def test_a_torch_without_cuda_imports_the_operators_and_they_refuse_its_tensors():
    child("import torch\n"
          "for name in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
          "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
          "from meganeura_b200 import ops\n"
          "try: ops.token_probs(torch.zeros(2, 8))\n"
          "except ValueError: pass\n"
          "else: raise SystemExit(1)\n")
