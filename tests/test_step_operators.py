"""What the operators around a step's shared layers refuse, before anything reaches a GPU."""
import pytest
import torch

from cubic_serve_b200.ops import kernels as K

I32 = torch.int32


def _ints(n, v=1):
    return torch.full((n,), v, dtype=I32)


def _layout_args(n=3, **kw):
    a = dict(request=torch.arange(n, dtype=I32), start=_ints(n), count=_ints(n), held=_ints(n), pages=_ints(n), table=torch.zeros(8, 4, dtype=I32),
             out=K.StepLayout(16, 8, 16, "cpu"), block=4, tokens=3, blocks=3, pad=0)
    a.update(kw)
    return a


@pytest.mark.parametrize("change", [
    dict(start=torch.ones(3)), dict(request=torch.ones(3, dtype=torch.int64)), dict(count=_ints(2)), dict(held=_ints(2)), dict(pages=torch.ones(2, 2, dtype=I32)),
    dict(start=torch.ones(6, dtype=I32)[::2]), dict(table=torch.zeros(8, 4)), dict(table=torch.zeros(8, 8, dtype=I32)[:, ::2]), dict(tokens=17), dict(blocks=17),
    dict(pad=17), dict(block=0), dict(block=1 << 21), dict(tokens=-1), dict(),
])
def test_step_layout_refuses(change):
    if "start" in change and change["start"].numel() == 6:
        change["start"] = change["start"][:3]
    with pytest.raises(ValueError):
        K.step_layout(**_layout_args(**change))


def test_step_layout_holds_a_limited_number_of_requests():
    with pytest.raises(ValueError):
        K.StepLayout(16, 5000, 16, "cpu")
    with pytest.raises(ValueError):
        K.step_layout(**_layout_args(n=9))
    with pytest.raises(ValueError):
        K.StepLayout(16, 8, 16, "cpu", into={"other": _ints(3)})
    with pytest.raises(ValueError):
        K.StepLayout(16, 8, 16, "cpu", into={"slots": _ints(3)})


def _bank(slots=2, k=64, n=96, rank=16, sections=1, dtype=torch.bfloat16, **kw):
    return K.AdapterBank(torch.zeros(slots, sections * rank, k, dtype=dtype), torch.zeros(slots, n, rank, dtype=dtype), torch.ones(slots), **kw)


@pytest.mark.parametrize("make", [
    lambda: _bank(dtype=torch.float16), lambda: _bank(rank=129), lambda: _bank(k=60), lambda: _bank(n=100), lambda: _bank(widths=(64, 64)), lambda: _bank(sections=2, widths=(40, 56)),
    lambda: _bank(sections=2, widths=(96,)), lambda: _bank(slots=1024), lambda: _bank(sections=5, n=160, widths=(32,) * 5), lambda: _bank(ranks=torch.ones(2)),
    lambda: K.AdapterBank(torch.zeros(2, 16, 64).bfloat16(), torch.zeros(3, 96, 16).bfloat16(), torch.ones(2)),
    lambda: K.AdapterBank(torch.zeros(2, 16, 64).bfloat16(), torch.zeros(2, 96, 16).bfloat16(), torch.ones(3)),
    lambda: K.AdapterRows(65536, 2, 16, "cpu"), lambda: K.AdapterRows(16, 1024, 16, "cpu"), lambda: K.AdapterRows(0, 4, 16, "cpu"),
])
def test_adapter_banks_refuse(make):
    with pytest.raises(ValueError):
        make()


def _stored(bank):
    """[slots, sections, stored ranks, k stored] of a bank's A."""
    return bank.a.transpose(1, 2).reshape(bank.slots, bank.sections, bank.rank, -1)


def test_bank_ranks_are_stored_as_the_next_width():
    b = _bank(rank=20, sections=3, n=96, widths=(32, 32, 32))
    assert b.rank == 32 and b.a.shape == (2, 2, 96, 32) and b.b.shape == (2, 96, 32) and b.ranks.tolist() == [20, 20]
    a = torch.randn(2, 3 * 20, 72).bfloat16()
    b = K.AdapterBank(a, torch.randn(2, 96, 20).bfloat16(), torch.ones(2), (32, 32, 32))
    assert torch.equal(_stored(b)[:, :, :20, :72].reshape(2, 60, 72), a) and not _stored(b)[:, :, 20:].any() and not _stored(b)[..., 72:].any()
    b.load(1, [torch.ones(4, 72), None, torch.full((20, 72), 2.0)], [torch.ones(32, 4), None, torch.ones(32, 20)], 0.5)
    s = _stored(b)[1]
    assert b.ranks.tolist() == [20, 20] and b.scale.tolist() == [1.0, 0.5] and not s[1].any() and s[0, :4, :72].eq(1).all() and not s[0, 4:].any() and s[2, :20, :72].eq(2).all()
    b.load(0, [torch.ones(3, 72)] * 3, [torch.ones(32, 3)] * 3, 1.0)
    assert b.ranks.tolist() == [3, 20]
    for bad in (dict(slot=2), dict(a=[torch.ones(21, 72), None, None], b=[torch.ones(32, 21), None, None]), dict(a=[torch.ones(4, 64)] * 3, b=[torch.ones(32, 4)] * 3), dict(a=[None] * 2, b=[None] * 2)):
        with pytest.raises(ValueError):
            b.load(**{"slot": 0, "a": [None] * 3, "b": [None] * 3, "scale": 1.0, **bad})


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(4, 64)), dict(x=torch.zeros(4, 56).bfloat16()), dict(x=torch.zeros(3, 64).bfloat16()), dict(y=torch.zeros(4, 88).bfloat16()),
    dict(y=torch.zeros(4, 100).bfloat16()[:, :96]), dict(out=torch.zeros(4, 96)), dict(x=torch.zeros(64, 4).bfloat16().t()), dict(rows=K.AdapterRows(4, 3, 16, "cpu")),
    dict(y=torch.zeros(4, 104).bfloat16()[:, 4:100]), dict(),
])
def test_adapter_add_refuses(change):
    rows = K.AdapterRows(4, 2, 16, "cpu")
    a = dict(x=torch.zeros(4, 64).bfloat16(), y=torch.zeros(4, 96).bfloat16(), bank=_bank(), rows=rows)
    a.update(change)
    a["rows"].rows = 4
    with pytest.raises(ValueError):
        K.adapter_add(**a)


def test_adapter_rows_refuse():
    with pytest.raises(ValueError):
        K.adapter_rows(_ints(5), K.AdapterRows(4, 2, 16, "cpu"))
    with pytest.raises(ValueError):
        K.adapter_rows(torch.zeros(4), K.AdapterRows(4, 2, 16, "cpu"))
    with pytest.raises(ValueError):
        K.adapter_rows(_ints(4), K.AdapterRows(4, 2, 16, "cpu"))           # not on a GPU


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(2, 9).half()), dict(logits=torch.zeros(9)), dict(vocab=10), dict(vocab=0), dict(out_ids=torch.zeros(2)), dict(out_ids=_ints(1)), dict(temperature=_ints(2)),
    dict(top_k=torch.zeros(2)), dict(top_p=torch.zeros(1)), dict(min_p=torch.zeros(2).double()), dict(uniforms=torch.zeros(2).half()), dict(seeds=_ints(2)), dict(mask=torch.zeros(2, 1)),
    dict(mask=torch.zeros(1, 1, dtype=I32)), dict(logits=torch.zeros(9, 2).t()), dict(logits=torch.zeros(2, 40), mask=torch.zeros(2, 1, dtype=I32)), dict(logits=torch.zeros(1, 9).expand(2, 9)),
    dict(rows=torch.zeros(2)), dict(),
])
def test_sample_vocabulary_refuses(change):
    a = dict(logits=torch.zeros(2, 9), out_ids=_ints(2), temperature=torch.ones(2))
    a.update(change)
    with pytest.raises(ValueError):
        K.sample_vocabulary(**a)


def test_calls_that_would_mean_something_else_are_refused():
    """A product that reads what it has written already; a draw without a number to draw with."""
    square = K.AdapterBank(torch.zeros(2, 16, 64).bfloat16(), torch.zeros(2, 64, 16).bfloat16(), torch.ones(2))
    rows = K.AdapterRows(4, 2, 16, "cpu")
    rows.rows = 4
    x, y = torch.zeros(4, 64).bfloat16(), torch.zeros(4, 64).bfloat16()
    with pytest.raises(ValueError, match="other memory"):
        K.adapter_add(x, x, square, rows)
    with pytest.raises(ValueError, match="other memory"):
        K.adapter_add(x, y, square, rows, out=x)
    with pytest.raises(ValueError, match="needs uniforms, or seeds"):
        K.sample_vocabulary(torch.zeros(2, 9), _ints(2), torch.ones(2))
