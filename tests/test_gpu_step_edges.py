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


_LAY = """
import sys, torch
from cubic_serve_b200.ops import kernels as K
n = int(sys.argv[1])
i = torch.arange(n, dtype=torch.int32, device="cuda")
table, start, one = (i[:, None] * 3 + torch.arange(3, dtype=torch.int32, device="cuda")).contiguous(), i % 40, torch.ones_like(i)
lay = K.step_layout(i, start, one, torch.full_like(i, 3), i[:0], table, K.StepLayout(n, n, n, "cuda"), 4, tokens=n, blocks=n)
assert lay.totals.tolist() == [n, n, 0, 0] and torch.equal(lay.row0, i) and torch.equal(lay.slots, (i * 3 + start // 16) * 16 + start % 16)
"""


@pytest.mark.parametrize("n", [2043, 2047])
def test_layouts_of_any_number_of_requests(n):
    """Sums of 48 KB less a little: more than 48 KB with the kernel's other shared memory."""
    _alone(_LAY, n)
