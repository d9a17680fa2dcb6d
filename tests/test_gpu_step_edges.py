"""Edges of the operators around a step's shared layers."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def _alone(code, *args):
    """In a process of its own: no larger size has run there before."""
    r = subprocess.run([sys.executable, "-c", code, *map(str, args)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


_SORT = """
import sys, torch
from cubic_serve_b200.ops import kernels as K
slots = int(sys.argv[1])
ids = (torch.arange(900, dtype=torch.int32, device="cuda") * 37) % (slots + 1) - 1
plan = K.adapter_rows(ids, K.AdapterRows(900, slots, 16, "cuda"))
key = torch.where(ids < 0, slots, ids.long())
assert torch.equal(plan.order.long(), torch.sort(key, stable=True).indices), "rows by adapter, by index among an adapter's"
"""


@pytest.mark.parametrize("slots", [568, 767])
def test_rows_are_sorted_over_any_number_of_slots(slots):
    """Tables of 36 to 48 KB: more than 48 KB with the kernel's other shared memory."""
    _alone(_SORT, slots)
