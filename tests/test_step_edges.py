"""Edges of the operators around a step's shared layers that need no GPU."""
import pytest
import torch

from cubic_serve_b200.ops import kernels as K


def test_a_refused_load_leaves_the_slot_as_it_was():
    """The second section's matrix is too wide: the first one's is not written either."""
    torch.manual_seed(0)
    bank = K.AdapterBank(torch.randn(2, 2 * 8, 64).bfloat16(), torch.randn(2, 64, 8).bfloat16(), torch.ones(2), (32, 32))
    held = [t.clone() for t in (bank.a, bank.b, bank.scale, bank.ranks, bank._section_ranks)]
    good_a, good_b = torch.ones(4, 64), torch.ones(32, 4)
    for a, b in (((good_a, torch.ones(9, 64)), (good_b, torch.ones(32, 9))), ((good_a, good_a), (good_b, torch.ones(31, 4))), ((good_a, None), (good_b, good_b)),
                 ((good_a, torch.ones(4)), (good_b, good_b)), ((good_a, good_a), (good_b, torch.ones(32)))):
        with pytest.raises(ValueError):
            bank.load(0, a, b, 3.0)
        assert all(torch.equal(t, h) for t, h in zip((bank.a, bank.b, bank.scale, bank.ranks, bank._section_ranks), held))


def test_ranks_that_are_not_in_use_may_hold_anything():
    """A bank over buffers that were never filled: what is behind the ranks in use is zero in B, so that no product makes NaN of it."""
    b = torch.full((3, 64, 24), float("nan")).bfloat16()
    b[0], b[1, :, :5] = 1, 2
    bank = K.AdapterBank(torch.full((3, 24, 64), float("nan")).bfloat16(), b, torch.full((3,), float("nan")), ranks=torch.tensor([24, 5, 0], dtype=torch.int32))
    assert bank.b[0, :, :24].eq(1).all() and bank.b[1, :, :5].eq(2).all() and not bank.b[0, :, 24:].any() and not bank.b[1, :, 5:].any() and not bank.b[2].any()
    assert b[2].isnan().all(), "the caller's is as it was"
