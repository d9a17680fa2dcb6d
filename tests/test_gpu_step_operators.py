"""The operators around a step's shared layers against plain forms in 64 bits: layout, adapters, draws from a whole vocabulary."""
import math

import numpy as np
import pytest
import torch

from cubic_serve_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32


# ------------------------------------------------------------------------------------------------- layout
def _plain_layout(request, start, count, held, pages, table, block, pad):
    """Python integers, one token at a time."""
    table = table.copy()
    out = {k: [] for k in ("positions", "slots", "rb_req", "rb_qstart", "rb_qcount", "rb_ctx", "row0", "logit_rows")}
    taken = 0
    for r, s, c, h in zip(request, start, count, held):
        for pg in range(h, -(-(s + c) // 16)):
            table[r, pg] = pages[taken]
            taken += 1
        row0 = len(out["positions"])
        out["row0"].append(row0)
        out["logit_rows"].append(row0 + c - 1 if c else -1)
        for j in range(c):
            out["positions"].append(s + j)
            page = int(table[r, (s + j) // 16])
            out["slots"].append(page * 16 + (s + j) % 16 if page >= 0 else -1)
        for f in range(0, c, block):
            for k, v in (("rb_req", r), ("rb_qstart", row0 + f), ("rb_qcount", min(block, c - f)), ("rb_ctx", s + f + 1)):
                out[k].append(v)
    totals = [len(out["positions"]), len(out["rb_req"]), taken, 0]
    while len(out["positions"]) < pad:
        out["positions"].append(0)
        out["slots"].append(-1)
    while len(out["rb_req"]) < pad:
        for k, v in (("rb_req", 0), ("rb_qstart", len(out["rb_qstart"])), ("rb_qcount", 0), ("rb_ctx", 0)):
            out[k].append(v)
    return out, table, totals


def _lay(n, most_start, most_count, block, pad=0, seed=0, width_extra=0, extra_pages=0, known=True, ahead=True):
    r = np.random.default_rng(seed)
    start, count = r.integers(0, most_start + 1, n), r.integers(0, most_count + 1, n)
    held = -(-start // 16) + (r.integers(0, 3, n) if ahead and known else 0)
    rows, width = n + 3, int(max(1, (-(-(start + count) // 16)).max(initial=0), held.max(initial=0))) + width_extra
    ids = r.permutation(rows * width + 9999)
    table = np.where(np.arange(width) < np.zeros((rows, 1)), 0, -1).astype(np.int32)
    req = r.permutation(rows)[:n]
    for i, q in enumerate(req):
        table[q, :held[i]] = ids[i * width:i * width + held[i]]
    need = np.maximum(0, -(-(start + count) // 16) - held)
    pages = ids[rows * width:rows * width + int(need.sum()) + extra_pages]
    want, want_table, totals = _plain_layout(req.tolist(), start.tolist(), count.tolist(), held.tolist(), pages.tolist(), table, block, pad)
    t, b = totals[0], totals[1]
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(DEV)        # noqa: E731
    wide = torch.full((rows, width + 5), -7, dtype=I32, device=DEV)                          # a table inside a wider one
    wide[:, :width] = cu(table)
    lay = K.StepLayout(max(t, pad) + 11, min(n + 2, 4096), max(b, pad) + 11, DEV)
    lay.totals.fill_(-77)
    for k in want:
        getattr(lay, k).fill_(-77)
    K.step_layout(cu(req), cu(start), cu(count), cu(held) if known else None, cu(pages), wide[:, :width], lay, block, tokens=t, blocks=b, pad=pad)
    for k, v in want.items():
        got = getattr(lay, k).cpu().tolist()
        assert got[:len(v)] == v, k
        assert all(g == -77 for g in got[len(v):]), f"{k}: rows behind the last one stay"
    assert torch.equal(wide[:, :width].cpu(), torch.from_numpy(want_table)) and bool((wide[:, width:] == -7).all())
    assert lay.totals.tolist() == totals
    lay.check()


@pytest.mark.parametrize("n,start,count,block,pad", [
    (1, 0, 1, 4, 0), (1, 15, 1, 4, 8), (1, 16, 17, 1, 0), (7, 100, 1, 4, 8), (256, 1300, 1, 4, 256), (37, 2000, 400, 4, 0), (3, 0, 4000, 16, 0), (300, 8000, 300, 2, 0), (5, 50, 0, 4, 0),
    (5, 50, 0, 4, 6), (4096, 300, 3, 8, 0), (1000, 64, 40, 3, 0), (513, 5, 1, 4, 1024),
])
def test_layout_equals_the_plain_form(n, start, count, block, pad):
    _lay(n, start, count, block, pad, seed=n + start)


def test_layout_takes_held_from_the_lengths_and_leaves_pages_over():
    _lay(9, 200, 90, 4, seed=5, known=False, extra_pages=4, width_extra=2)
    _lay(0, 0, 0, 4, pad=4)
    _lay(0, 0, 0, 4, pad=0)


def test_layout_refuses_on_the_device_what_it_cannot_place():
    """Too few pages, too long, a row that is not there, more rows than there is room for: in bounds, no slots, and said."""
    cu = lambda *a: torch.tensor(a, dtype=I32, device=DEV)        # noqa: E731
    table = torch.full((4, 3), -1, dtype=I32, device=DEV)
    table[0, 0] = 40
    guard = table.clone()
    lay = K.StepLayout(64, 4, 64, DEV)
    K.step_layout(cu(0, 7, 1, -1), cu(10, 0, 40, 5), cu(4, 3, 20, 1), cu(1, 0, 3, 1), cu(50), table, lay, 4, tokens=28, blocks=8)
    assert lay.slots[:28].tolist() == [650, 651, 652, 653] + [-1] * 24 and lay.totals.tolist() == [28, 8, 0, 6]
    assert lay.rb_qcount[:8].tolist() == [4] + [0] * 7 and lay.rb_req[:8].tolist() == [0] * 8 and torch.equal(table, guard)
    with pytest.raises(RuntimeError, match="longer than the block table.*does not have"):
        lay.check()
    K.step_layout(cu(0, 1), cu(10, 0), cu(4, 40), cu(1, 0), cu(60, 61), table, lay, 8, tokens=44, blocks=6)
    assert lay.slots[:44].tolist() == [650, 651, 652, 653] + [960 + i for i in range(32)] + [-1] * 8 and lay.totals.tolist() == [44, 6, 3, 1]
    assert lay.rb_qcount[:6].tolist() == [4, 0, 0, 0, 0, 0], "a request that lacks pages attends to nothing"
    assert table[1].tolist() == [60, 61, -1]
    lay.slots.fill_(-5)
    K.step_layout(cu(0, 1), cu(10, 0), cu(4, 20), cu(1, 2), cu(9), table, lay, 4, tokens=6, blocks=2)
    assert lay.slots[:6].tolist() == [650, 651, 652, 653, 960, 961] and lay.slots[6:].eq(-5).all() and lay.totals.tolist() == [24, 6, 0, 8]
    assert lay.rb_qcount[:2].tolist() == [4, 0] and lay.logit_rows[:2].tolist() == [3, -1]
    huge = 2 ** 31 - 1
    K.step_layout(cu(0, 1, 2), cu(huge, 10, 3), cu(huge, huge, -4), cu(-3, huge, 0), cu(9), table, lay, 4, tokens=64, blocks=16)
    assert lay.slots.eq(-1).all() and lay.rb_qcount[:16].eq(0).all() and lay.totals[3].item() & 2


def test_layout_in_a_graph_and_on_another_stream():
    r = np.random.default_rng(0)
    n, width = 64, 90
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        start, count = torch.from_numpy(r.integers(0, 1300, n).astype(np.int32)).to(DEV), torch.ones(n, dtype=I32, device=DEV)
        table = torch.from_numpy(r.permutation(n * width).reshape(n, width).astype(np.int32)).to(DEV)
        req, pages, lay = torch.arange(n, dtype=I32, device=DEV), torch.arange(n, dtype=I32, device=DEV) + n * width, K.StepLayout(n, n, n, DEV)
        run = lambda: K.step_layout(req, start, count, None, pages, table, lay, 4, tokens=n, blocks=n, pad=n)        # noqa: E731
        run()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            run()
        for step in range(40):
            g.replay()
            st.synchronize()
            t, s = table.cpu().numpy(), start.cpu().numpy()
            assert lay.slots.tolist() == [int(t[i, s[i] // 16]) * 16 + int(s[i]) % 16 for i in range(n)]
            start += 1


# ------------------------------------------------------------------------------------------------- adapters
def _adapter_case(rows, slots, rank, k, widths, ids, seed=0, ranks=None, pad_x=0, pad_y=0, scale_x=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s, std: torch.randn(*s, device=DEV, generator=g) * std        # noqa: E731
    n, S = sum(widths), len(widths)
    x, y = rnd(rows, k + pad_x, std=scale_x).bfloat16()[:, :k], rnd(rows, n + pad_y, std=1.0).bfloat16()[:, :n]
    a, b = rnd(slots, S * rank, k, std=k ** -0.5).bfloat16(), rnd(slots, n, rank, std=0.3).bfloat16()
    scale = torch.rand(slots, device=DEV, generator=g) + 0.5
    return x, y, a, b, scale


def _adapter_truth(x, y, a, b, scale, widths, ids, ranks=None):
    """The sum in 64 bits, and what the result may be off: half a step of bf16, 2^-16 of every h by its two parts, fp32 sums of k and of
    the ranks (two roundings a term at most)."""
    out, err = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=y.device)
    k, rank = x.shape[1], b.shape[2]
    for t, s in enumerate(ids.tolist()):
        if not 0 <= s < a.shape[0]:
            continue
        r = rank if ranks is None else int(ranks[s])
        col = 0
        for i, w in enumerate(widths):
            A, B = a[s, i * rank:i * rank + r].double(), b[s, col:col + w, :r].double()
            h, size = A @ x[t].double(), A.abs() @ x[t].double().abs()
            out[t, col:col + w] += scale[s].double() * (B @ h)
            err[t, col:col + w] = scale[s].double() * (B.abs() @ (h.abs() * 2.0 ** -16 + size * 2.0 ** -23 * (k + 8))) + scale[s].double() * (B.abs() @ h.abs()) * 2.0 ** -23 * (2 * rank + 4)
            col += w
    err += (out.abs() + err) * 2.0 ** -8
    return out, err


def _check_adapter(rows, slots, rank, k, widths, ids, seed=0, ranks=None, in_place=False, pad_x=0, pad_y=0):
    x, y, a, b, scale = _adapter_case(rows, slots, rank, k, widths, ids, seed, ranks, pad_x, pad_y)
    bank = K.AdapterBank(a, b, scale, widths, ranks=None if ranks is None else torch.tensor(ranks, dtype=I32, device=DEV))
    plan = K.AdapterRows(rows, slots, len(widths) * rank, DEV)
    want, err = _adapter_truth(x, y, a, b, scale, widths, ids, ranks)
    before = y.clone()
    K.adapter_rows(torch.tensor(ids.tolist(), dtype=I32, device=DEV), plan)
    out = y if in_place else torch.full((rows, y.shape[1] + 8), 7.0, device=DEV).bfloat16()[:, :y.shape[1]]
    K.adapter_add(x, y, bank, plan, out=None if in_place else out)
    off = (out.double() - want).abs() - err
    assert not bool((off > 0).any()), float(off.max())
    none = [t for t, s in enumerate(ids.tolist()) if not 0 <= s < slots]
    assert torch.equal(out[none], before[none])
    return out


@pytest.mark.parametrize("rows,slots,rank,k,widths", [
    (1, 1, 16, 128, (64,)), (1, 8, 16, 4096, (512, 128, 128)), (3, 2, 8, 72, (40,)), (17, 3, 20, 200, (32, 96, 8)), (48, 16, 32, 1024, (256, 256)), (64, 64, 64, 520, (1024,)),
    (65, 1, 16, 64, (264,)), (130, 4, 128, 640, (96, 32)), (257, 5, 16, 1032, (160, 64, 64, 32)), (300, 7, 48, 336, (288,)), (700, 3, 16, 512, (520,)), (2, 1023, 16, 16, (8,)),
    (1100, 300, 16, 64, (32, 32)),
])
def test_adapters_against_64_bits(rows, slots, rank, k, widths):
    g = np.random.default_rng(rows + slots)
    ids = g.integers(-1, slots + 1, rows)                          # -1 and a slot that there is not: none
    _check_adapter(rows, slots, rank, k, widths, ids, seed=rows)


@pytest.mark.parametrize("layout", ["one", "none", "sorted", "alternating", "last"])
def test_adapters_by_how_rows_share_them(layout):
    rows, slots = 210, 6
    ids = {"one": np.full(rows, 3), "none": np.full(rows, -1), "sorted": np.arange(rows) * slots // rows, "alternating": np.arange(rows) % slots, "last": np.where(np.arange(rows) == rows - 1, 5, -1)}[layout]
    a = _check_adapter(rows, slots, 16, 264, (64, 64), ids, seed=1)
    b = _check_adapter(rows, slots, 16, 264, (64, 64), ids, seed=1, in_place=True)
    assert torch.equal(a, b)


def test_adapter_rows_of_strided_inputs_and_ranks_in_use():
    ids = np.array([0, 1, 2, 3, -1] * 9)
    _check_adapter(45, 4, 64, 320, (96, 64), ids, ranks=[64, 0, 5, 33], pad_x=24, pad_y=40)
    _check_adapter(45, 4, 16, 320, (96, 64), ids, ranks=[0, 0, 0, 0], pad_x=8, pad_y=8, in_place=True)


def test_what_is_not_finite_stays_in_its_row():
    """An infinity or NaN in one row's x or y reaches that row alone, and an infinity meets no zero of the stored ranks."""
    rows, k, n = 40, 256, 64
    x, y, a, b, scale = _adapter_case(rows, 2, 20, k, (n,), None, seed=3)
    ids = torch.arange(rows, dtype=I32, device=DEV) % 2
    plan = K.adapter_rows(ids, K.AdapterRows(rows, 2, 20, DEV))
    bank = K.AdapterBank(a.abs() + 0.01, b.abs() + 0.01, scale, (n,))
    clean = K.adapter_add(x, y, bank, plan, out=torch.empty_like(y))
    x2, y2 = x.clone(), y.clone()
    x2[5, 7], x2[6, 9], x2[7, 0], y2[8, 3] = math.inf, math.nan, -math.inf, math.inf
    got = K.adapter_add(x2, y2, bank, plan, out=torch.empty_like(y))
    keep = [t for t in range(rows) if t not in (5, 6, 7, 8)]
    assert torch.equal(got[keep], clean[keep]) and bool((got[5] == math.inf).all()) and bool(got[6].isnan().all()) and bool((got[7] == -math.inf).all())
    assert got[8, 3] == math.inf and torch.equal(got[8, :3], clean[8, :3]) and torch.equal(got[8, 4:], clean[8, 4:])


def test_a_row_does_not_depend_on_its_neighbours():
    """The same row alone, among others of its adapter and among other adapters: the same bits, and twice the same step too."""
    x, y, a, b, scale = _adapter_case(129, 4, 32, 768, (128, 64), None, seed=9)
    bank, plan = K.AdapterBank(a, b, scale, (128, 64)), K.AdapterRows(129, 4, 64, DEV)
    ids = torch.randint(-1, 4, (129,), generator=torch.Generator().manual_seed(0)).to(I32).to(DEV)
    K.adapter_rows(ids, plan)
    first = K.adapter_add(x, y, bank, plan, out=torch.empty_like(y))
    assert torch.equal(first, K.adapter_add(x, y, bank, plan, out=torch.empty_like(y)))


def test_adapters_in_a_graph_follow_the_ids_and_the_weights():
    """A captured step replays with other ids, another slot's weights and other rows; the plan of a second graph is its own."""
    rows, k, widths = 24, 512, (96, 32)
    x, y, a, b, scale = _adapter_case(rows, 3, 16, k, widths, None, seed=4)
    bank = K.AdapterBank(a, b, scale, widths)
    graphs = []
    for _ in range(2):
        ids, out, plan = torch.zeros(rows, dtype=I32, device=DEV), torch.empty(rows, 128, device=DEV, dtype=torch.bfloat16), K.AdapterRows(rows, 3, 32, DEV)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            K.adapter_add(x, y, bank, K.adapter_rows(ids, plan), out=out)
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                K.adapter_add(x, y, bank, K.adapter_rows(ids, plan), out=out)
        graphs.append((g, ids, out, st))
    for trial in range(3):
        new_a, new_b = [torch.randn(16, k, device=DEV).bfloat16() * 0.05 for _ in widths], [torch.randn(n, 16, device=DEV).bfloat16() * 0.1 for n in widths]
        bank.load(trial % 3, new_a, new_b, 0.5 + trial)
        a[trial % 3], b[trial % 3], scale[trial % 3] = torch.cat(new_a), torch.cat(new_b), 0.5 + trial
        for i, (g, ids, out, st) in enumerate(graphs):
            ids.copy_(torch.from_numpy(np.random.default_rng(10 * trial + i).integers(-1, 3, rows).astype(np.int32)))
        torch.cuda.synchronize()
        for g, _, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for g, ids, out, _ in graphs:
            want, err = _adapter_truth(x, y, a, b, scale, widths, ids)
            assert bool(((out.double() - want).abs() <= err).all())


# ------------------------------------------------------------------------------------------------- draws
def _plain_draw(x, t, k, p, m, u, mask=None):
    """(id, log-probability, tokens kept) of one row, float64 numpy."""
    x = x.astype(np.float64)
    ids = np.arange(len(x))
    ok = (x == x) & (x > -np.inf)
    if mask is not None:
        ok &= (mask[ids >> 5] >> (ids & 31) & 1).astype(bool)
    ids = ids[ok]
    if not len(ids):
        return 0, -math.inf, 0
    ids = ids[np.argsort(-x[ids], kind="stable")]
    if not t > 0:
        return int(ids[0]), 0.0, 1
    v, n = x[ids], len(ids)
    with np.errstate(all="ignore"):
        w = np.where(v == v[0], 1.0, 0.0 if v[0] == np.inf else np.exp((v - v[0]) / t))          # beside an infinity nothing else has weight
    if k > 0:
        n = min(n, k)
    upto = np.cumsum(w)
    if p < 1:
        n = min(n, 1 + int((upto[:n] < max(p, 0.0) * upto[n - 1]).sum()))
    if m >= 2.0 ** -60:
        n = min(n, max(1, int((w >= min(m, 1.0)).sum())))
    pick = min(int((upto[:n] <= u * upto[n - 1]).sum()), n - 1)
    return int(ids[pick]), math.log(w[pick] / upto[n - 1]), n


def _check_draw(x, t=1.0, k=0, p=1.0, m=0.0, u=0.5, mask=None, seed=None):
    """``x`` [rows, vocab] on the GPU; settings are numbers or a list, one a row."""
    rows, vocab = x.shape
    full = lambda v, dt: torch.tensor([v] * rows if not isinstance(v, (list, np.ndarray)) else list(v), dtype=dt, device=DEV)        # noqa: E731
    t, k, p, m, u = full(t, torch.float32), full(k, I32), full(p, torch.float32), full(m, torch.float32), full(u, torch.float32)
    ids, lp, kept = torch.full((rows,), -9, dtype=I32, device=DEV), torch.zeros(rows, device=DEV), torch.zeros(rows, dtype=I32, device=DEV)
    K.sample_vocabulary(x, ids, t, k, p, m, uniforms=u, mask=mask, out_logprob=lp, out_kept=kept)
    h = [v.double().cpu().numpy() for v in (t, k, p, m, u)]
    xs, mk = x.float().cpu().numpy(), None if mask is None else mask.cpu().numpy().view(np.uint32)
    for r in range(rows):
        want = _plain_draw(xs[r], h[0][r], int(h[1][r]), h[2][r], h[3][r], h[4][r], None if mk is None else mk[r])
        got = (int(ids[r]), float(lp[r]), int(kept[r]))
        assert (got[0], got[2]) == (want[0], want[2]), (r, got, want)
        # one rounding to fp32, and masses in units of 2^-42: half a unit a token
        assert got[1] == want[1] or abs(got[1] - want[1]) <= abs(want[1]) * 2.0 ** -24 + vocab * 2.0 ** -43 + 1e-12, (r, got, want)


def _logits(rows, vocab, dtype, seed=0, std=2.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, vocab, device=DEV, generator=g) * std
    hot = torch.randint(0, vocab, (rows, 5), device=DEV, generator=g)
    x[torch.arange(rows, device=DEV)[:, None], hot] += 8.0
    return x.to(dtype)


DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 257, 1000, 4099, 50257, 151936])
def test_draws_equal_the_plain_form(dtype, vocab):
    rows = 12
    r = np.random.default_rng(vocab)
    _check_draw(_logits(rows, vocab, dtype, vocab), t=r.choice([0.0, 0.3, 0.7, 1.0, 2.0], rows), k=r.choice([0, 1, 5, 20, 21, 100, 3000, 10 ** 9], rows),
                p=r.choice([1.0, 0.9, 0.5, 0.999, 0.01], rows), m=r.choice([0.0, 0.05, 0.3, 1e-6, 1.0], rows), u=r.random(rows))


@pytest.mark.parametrize("dtype", DTYPES)
def test_draws_over_the_whole_mass_and_each_filter_alone(dtype):
    rows, vocab = 16, 32003
    x = _logits(rows, vocab, dtype, 3)
    u = [(i + 0.37) / rows for i in range(rows)]
    for kw in (dict(), dict(t=1.7), dict(t=0.05), dict(k=1), dict(k=37), dict(k=vocab), dict(p=0.9), dict(p=0.0), dict(p=1e-30), dict(m=0.1), dict(m=1.0), dict(m=5.0), dict(m=1e-25), dict(t=0.0)):
        _check_draw(x, u=u, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.25, 0.5, 0.75, 1 - 2.0 ** -24])
def test_draws_among_equal_values_take_the_lowest_id(dtype, u):
    """Every logit the same; then four values in turn.  Prefixes end inside runs of equal values."""
    _check_draw(torch.full((1, 1024), 1.5, device=DEV, dtype=dtype), u=u)
    _check_draw(torch.zeros(2, 4096, device=DEV, dtype=dtype), u=u, k=[64, 0], p=[0.5, 0.25])
    x = (torch.arange(1000, device=DEV) % 4).to(dtype).expand(3, 1000).contiguous()
    _check_draw(x, u=u, k=[300, 0, 251], p=[1.0, 0.7, 0.93], t=[1.0, 0.5, 3.0])
    _check_draw(-x, u=u, k=[300, 0, 251], p=[1.0, 0.7, 0.93], t=[1.0, 0.5, 3.0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_draws_with_values_at_the_ends(dtype):
    """Both infinities, NaN, both zeros, the largest and the smallest magnitudes, temperatures from 1e-20 to infinity."""
    rows = 9
    base = _logits(rows, 3000, dtype, 8)
    u, t = [(i + 0.5) / rows for i in range(rows)], [1e-20, 1e-3, 0.02, 0.3, 1.0, 30.0, 4e4, 1e20, math.inf]
    _check_draw(base, t=t, u=u)
    for fill in ((0, math.inf), (1, -math.inf), (2, math.nan)):
        x = base.clone()
        x[:, 17::(50 if fill[0] else 1000)] = fill[1]
        _check_draw(x, t=t, u=u, k=[0, 2, 0, 7, 0, 500, 0, 9, 0])
        _check_draw(x, t=t, u=u, p=0.8, m=[0.0, 0.0, 0.1, 0.1, 0.1, 0.5, 0.5, 0.5, 0.5])
    for size in (1e-38, 1e-30, 1e-12, 1e-4, 1e4, 1e9, 1e30):
        _check_draw((base.double() * size).to(dtype), t=t, u=u)
        _check_draw((base.double() * size).to(dtype), t=size, u=u, k=[0, 1, 100, 0, 9, 2000, 0, 5, 0], p=[1.0, 0.9, 1.0, 0.5, 0.9, 1.0, 0.99, 1.0, 0.3])
    x = torch.zeros(rows, 700, device=DEV, dtype=dtype)
    x[:, ::3] = -0.0
    x[:, 1::7] = 1e-20
    x[:, 2::11] = -1e-20
    _check_draw(x, u=u, t=1.0, k=[0, 1, 50, 101, 400, 650, 0, 0, 0], p=[1.0] * 6 + [0.1, 0.5, 0.9])
    _check_draw(torch.full((1, 50), -math.inf, device=DEV, dtype=dtype))
    _check_draw(torch.full((2, 50), math.nan, device=DEV, dtype=dtype), t=[0.0, 1.0])
    _check_draw(torch.full((2, 50), math.inf, device=DEV, dtype=dtype), t=[0.0, 1.0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [33, 1000, 50257])
def test_draws_under_masks(dtype, vocab):
    """A row that allows everything, a few, one token, none, and the last token alone; bits behind the vocabulary are set."""
    rows, words = 6, -(-vocab // 32)
    r = np.random.default_rng(2)
    bits = np.ones((rows, words * 32), dtype=bool)
    bits[1] = r.random(words * 32) < 0.02
    bits[1, 5] = True
    bits[2:5, :vocab] = False
    bits[2, 29] = True
    bits[4, vocab - 1] = True
    bits[5, :] = r.random(words * 32) < 0.5
    mask = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).to(DEV)
    x = _logits(rows, vocab, dtype, 4)
    for kw in (dict(), dict(k=3), dict(p=0.7), dict(m=0.2), dict(t=0.0)):
        _check_draw(x, u=0.61, mask=mask, **kw)
    wide = torch.zeros(rows, words + 3, dtype=I32, device=DEV)
    wide[:, 2:2 + words] = mask
    _check_draw(x, u=0.61, mask=wide[:, 2:2 + words], p=0.9)
    _check_draw(x, u=0.61, mask=mask[5:].expand(rows, words), p=0.9)         # one mask for all rows


@pytest.mark.parametrize("dtype", DTYPES)
def test_draws_of_rows_at_any_address(dtype):
    """Rows at odd offsets of a wider buffer whose other columns would win."""
    wide = torch.full((5, 3331), 90.0, device=DEV, dtype=dtype)
    for off in range(0, 9):
        view = wide[:, off:off + 3001]
        view.copy_(_logits(5, 3001, dtype, off))
        _check_draw(view, u=[0.1, 0.3, 0.5, 0.7, 0.9], k=[0, 40, 0, 0, 7], p=[1.0, 1.0, 0.8, 0.99, 1.0])
        wide.fill_(90.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 18, 37, 38, 74, 75, 149])
@pytest.mark.parametrize("vocab", [8192, 16400, 32801])
def test_draws_of_any_number_of_rows(dtype, rows, vocab):
    """Rows are shared by one, two, four and eight blocks, by how many there are and how long: every way draws the same."""
    x = _logits(rows, vocab, dtype, rows + vocab)
    x[1:] = x[:1]                                                              # equal rows draw the same for the same number
    one = torch.ones(rows, device=DEV)
    ids, alone = torch.full((rows,), -1, dtype=I32, device=DEV), torch.full((1,), -1, dtype=I32, device=DEV)
    for u in (0.03, 0.4, 0.97):
        K.sample_vocabulary(x, ids, one, top_p=one * 0.97, min_p=one * 1e-4, uniforms=one * u)
        K.sample_vocabulary(x[:1], alone, one, top_p=one * 0.97, min_p=one * 1e-4, uniforms=one * u)
        assert ids.eq(alone).all()
    _check_draw(x[:2], k=300, p=0.9, m=0.01, u=0.37)


def test_draws_with_narrow_bins():
    """fp32 values that share their upper sixteen bits, and runs of equal ones among them."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = 1.0 + torch.randint(0, 3000, (8, 20000), device=DEV, generator=g).float() * 2.0 ** -23
    _check_draw(x, t=[1.0, 1e-4, 1e-3, 0.1, 1.0, 1.0, 1.0, 1.0], u=[0.1, 0.9, 0.4, 0.2, 0.6, 0.7, 0.8, 0.99], k=[0, 0, 0, 0, 1, 77, 19999, 5000], p=[0.5, 1.0, 0.9, 1.0, 1.0, 1.0, 0.3, 1.0])


def test_draws_of_chosen_rows_leave_the_others():
    x = _logits(10, 5000, torch.bfloat16, 6)
    u = torch.rand(10, device=DEV)
    one = torch.ones(10, device=DEV)
    want, ids = torch.zeros(10, dtype=I32, device=DEV), torch.full((10,), -3, dtype=I32, device=DEV)
    K.sample_vocabulary(x, want, one, uniforms=u)
    K.sample_vocabulary(x, ids, one, uniforms=u, rows=torch.tensor([7, -1, 2, 10, 9, 2, 2 ** 31 - 1], dtype=I32, device=DEV))
    assert [int(v) for v in ids] == [int(want[i]) if i in (2, 7, 9) else -3 for i in range(10)]


def test_draws_agree_with_the_sampler_of_twenty_candidates():
    """Same stream, same candidates: the whole-vocabulary draw with top-k of at most 20 picks what ``sample`` picks (fp32 sums there: but for
    draws within 1e-5 of a border, of which 4000 hold about one)."""
    rows = 4000
    x = _logits(rows, 2000, torch.bfloat16, 11)
    full = lambda v, dt: torch.full((rows,), v, dtype=dt, device=DEV)        # noqa: E731
    seeds, ctr = torch.arange(rows, device=DEV, dtype=torch.int64) * 77 + 5, torch.arange(rows, device=DEV, dtype=torch.int64) % 9
    a, b = full(0, I32), full(0, I32)
    K.sample(x, a, temperature=full(0.8, torch.float32), top_p=full(0.93, torch.float32), top_k=full(20, I32), seeds=seeds, counters=ctr)
    K.sample_vocabulary(x, b, full(0.8, torch.float32), full(20, I32), full(0.93, torch.float32), seeds=seeds, counters=ctr)
    assert int((a != b).sum()) <= 4


def test_draws_follow_their_probabilities():
    """40000 draws of one row by the stream of seeds: every token's share within five standard deviations."""
    rows = 40000
    x = torch.tensor([1.0, 0.0, 2.0, -1.0, 0.5, 2.0, -30.0], device=DEV).bfloat16().expand(rows, 7).contiguous()
    ids = torch.zeros(rows, dtype=I32, device=DEV)
    K.sample_vocabulary(x, ids, torch.ones(rows, device=DEV), seeds=torch.arange(rows, device=DEV, dtype=torch.int64), counters=torch.zeros(rows, device=DEV, dtype=torch.int64))
    p = torch.softmax(x[0].double(), 0).cpu()
    n = torch.bincount(ids.long(), minlength=7).double().cpu()
    assert bool(((n - rows * p).abs() <= 5 * (rows * p * (1 - p)).sqrt() + 1).all()), (n, rows * p)


def test_draws_in_a_graph():
    x = _logits(5, 9001, torch.bfloat16, 2)
    u, t, ids = torch.zeros(5, device=DEV), torch.ones(5, device=DEV), torch.zeros(5, dtype=I32, device=DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        K.sample_vocabulary(x, ids, t, uniforms=u)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            K.sample_vocabulary(x, ids, t, uniforms=u)
        for trial in range(4):
            x.copy_(_logits(5, 9001, torch.bfloat16, 20 + trial))
            u.uniform_()
            g.replay()
            st.synchronize()
            xs, us = x.float().cpu().numpy(), u.double().cpu().numpy()
            assert ids.tolist() == [_plain_draw(xs[r], 1.0, 0, 1.0, 0.0, us[r])[0] for r in range(5)]
