"""Attention of trees of drafts, the logits that requests want and the end of a tree's round against plain forms in 64 bits."""
import numpy as np
import pytest
import torch

from cubic_serve_b200.ops import eager
from cubic_serve_b200.ops import kernels as K
from cubic_serve_b200.ops.native import NativeLibraryError
from cubic_serve_b200.runtime.trees import tree_masks

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32
D = 128
BITS = [(8, 8), (4, 8), (6, 6), (4, 4), (8, 4), (6, 8), (8, 6), (4, 6), (6, 4)]


def _i32(v):
    return torch.from_numpy(np.ascontiguousarray(v).astype(np.int32)).to(DEV)


def _parents(n, r, wide=4):
    return [-1] + [int(r.integers(max(0, j - wide), j)) for j in range(1, n)]


# ------------------------------------------------------------------------------------------------- attention
class _Round:
    """Requests with trees behind contexts: a cache of random codes (slots past a request's tokens hold NaN scales), queries and masks."""

    def __init__(self, sizes, hq, hkv, kb, vb, seed=0, masks=None, words=None, spread=1.0):
        r = np.random.default_rng(seed)
        self.sizes, self.hq, self.hkv, self.kb, self.vb = sizes, hq, hkv, kb, vb
        lay = eager.blob_layout(D, kb, vb)
        held = [-(-(s + c) // 16) for s, c in sizes]
        order = r.permutation(sum(held) + 2)
        self.slots = r.permutation(len(sizes) + 2)[:len(sizes)]
        table = np.full((len(sizes) + 2, max(held) + 1), -1)
        blob = torch.from_numpy(r.integers(0, 256, (sum(held) + 2, hkv, lay["bytes"]), dtype=np.uint8))
        at = 0
        for i, (s, c) in enumerate(sizes):
            for j in range(held[i]):
                page = table[self.slots[i], j] = order[at]
                at += 1
                for name, end, of, bits in (("k_scale", "v_code", 1.2, kb), ("v_scale", "bytes", 1.0, vb)):
                    scale = torch.from_numpy((r.random((hkv, 16, D // 32)) + 0.5).astype(np.float32)) * of * spread / (1 << (bits - 1))
                    scale[:, max(0, s + c - 16 * j):] = float("nan")
                    blob[page, :, lay[name]:lay[end]] = scale.reshape(hkv, -1).contiguous().view(torch.uint8).reshape(hkv, -1)
        self.cache, self.table = blob.to(DEV), _i32(table)
        rows = sum(c for _, c in sizes)
        self.row0 = np.concatenate([[0], np.cumsum([c for _, c in sizes])[:-1]]).astype(int)
        words = words or max(1, -(-max(c for _, c in sizes) // 32))
        self.sees = np.zeros((rows, words), dtype=np.uint32)
        for i, (_, c) in enumerate(sizes):
            if c:
                self.sees[self.row0[i]:self.row0[i] + c] = tree_masks(_parents(c, r), words) if masks is None else masks(c, words, r)
        self.q = torch.from_numpy(r.standard_normal((rows, hq * D)).astype(np.float32)).to(DEV).bfloat16()

    def scales(self):
        lay = eager.blob_layout(D, self.kb, self.vb)
        return [self.cache[:, :, lay[a]:lay[b]].view(torch.float32).view(*self.cache.shape[:2], 16, D // 32) for a, b in (("k_scale", "v_code"), ("v_scale", "bytes"))]

    def args(self):
        return (self.cache, self.table, _i32(self.slots), _i32(self.row0), _i32([c for _, c in self.sizes]), _i32([s for s, _ in self.sizes]),
                torch.from_numpy(self.sees.view(np.int32)).to(DEV), self.hq, self.hkv, D, self.kb, self.vb)

    def run(self, **kw):
        out = torch.full_like(self.q, 7.0)
        ws = K.Workspace(torch.device(DEV, 0), 16, 16, 16)
        K.tree_attention(self.q, out, *self.args(), ws=ws, **kw)
        ws.check_status()
        return out

    def truth(self, scale=D ** -0.5):
        """(result, how far a kernel may be off), in 64 bits.

        Keys and values are products of codes and scales that are rounded to f16 (2^-11 each), probabilities are rounded to f16, the result to bf16 (2^-8);
        a score is off by 2^-10 of the sum of its products' magnitudes at most, which moves a probability and its sum by as much; sums in 32 bits,
        exponentials and the sums of the matrix units add less than 2^-16.

        The largest scale lies between 2^-10 and 2^-9 in the unit of the operands, whose smallest steps are 2^-24; a product and the bias in it are each off by
        half of one at most, so that a key or value may be off by 2^-14 of the largest scale besides.

        A probability below 2^-14 has the absolute steps of f16's smallest numbers instead: it is off by half of one, 2^-25, at most, relative to a running
        maximum that is not above the row's own, so that the sum it is divided by is one at least: 2^-25 of the sum of the values' magnitudes."""
        ref, tol = torch.zeros(self.q.shape, dtype=torch.float64), torch.zeros(self.q.shape, dtype=torch.float64)
        cache, table, group = self.cache.cpu(), self.table.cpu(), self.hq // self.hkv
        for i, (s, c) in enumerate(self.sizes):
            if not c:
                continue
            rows = slice(self.row0[i], self.row0[i] + c)
            sees = torch.ones(c, s + c, dtype=torch.bool)
            bits = (self.sees[rows][:, :, None] >> np.arange(32, dtype=np.uint32)) & 1
            sees[:, s:] = torch.from_numpy(bits.reshape(c, -1)[:, :c].astype(bool))
            for h in range(self.hkv):
                pages = [eager.decode_cache_page(cache[p, h], D, self.kb, self.vb) for p in table[self.slots[i], :-(-(s + c) // 16)].tolist()]
                k, v = (torch.cat([page[x] for page in pages])[:s + c].double() for x in (0, 1))
                q = self.q[rows, h * group * D:(h + 1) * group * D].cpu().double().view(c, group, D)
                z = torch.einsum("cgd,td->cgt", q, k) * scale
                most = [torch.cat([self.scales()[x][p, h].flatten() for p in table[self.slots[i], :-(-(s + c) // 16)].tolist()]).nan_to_num().max().item() for x in (0, 1)]
                off = torch.einsum("cgd,td->cgt", q.abs(), k.abs()) * scale * 2.0 ** -10 + q.abs().sum(-1, keepdim=True) * scale * 2.0 ** -14 * most[0]
                z = z.masked_fill(~sees[:, None], -torch.inf)
                p = torch.where(sees[:, None], torch.exp(z - z.amax(-1, keepdim=True)), 0.0)
                sums = p.sum(-1, keepdim=True)
                p = torch.where(sums > 0, p / sums, 0.0)
                o, a = torch.einsum("cgt,td->cgd", p, v), torch.einsum("cgt,td->cgd", p, v.abs())
                e = torch.where(sees[:, None], off, 0.0).amax(-1, keepdim=True)
                t = (torch.expm1(2 * e) + 3 * 2.0 ** -11 + 2.0 ** -16) * a * 1.01 + 2.0 ** -14 * most[1] + 2.0 ** -8 * o.abs() + 2.0 ** -25 * torch.einsum("cgt,td->cgd", sees[:, None].double().expand(z.shape), v.abs())
                ref[rows, h * group * D:(h + 1) * group * D], tol[rows, h * group * D:(h + 1) * group * D] = o.reshape(c, -1), t.reshape(c, -1)
        return ref, tol

    def check(self, **kw):
        got = self.run(**kw)
        ref, tol = self.truth(**kw)
        off = (got.cpu().double() - ref).abs()
        assert torch.isfinite(got.float()).all() and bool((off <= tol + 1e-30).all()), f"off by {(off / (tol + 1e-30)).max():.3g} of what is allowed"
        return got


@pytest.mark.parametrize("kb,vb", BITS)
def test_attention_of_every_width(kb, vb):
    _Round([(37, 9), (0, 5), (130, 1), (64, 33)], 8, 2, kb, vb, seed=kb * 8 + vb).check()


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (6, 2), (14, 2), (7, 1), (16, 1), (40, 2), (128, 1)])
def test_attention_of_every_head_layout(hq, hkv):
    _Round([(50, 7), (3, 20), (200, 2)], hq, hkv, 8, 8, seed=hq).check()


@pytest.mark.parametrize("start", [0, 1, 15, 16, 17, 47, 48, 63, 64, 65, 100, 127, 128, 1000])
@pytest.mark.parametrize("count", [1, 2, 16, 31, 33, 64, 65, 100, 129, 256])
def test_attention_of_lengths(start, count):
    _Round([(start, count)], 2, 1, 8, 8, seed=start + 1000 * count).check()


def test_attention_of_many_requests():
    r = np.random.default_rng(5)
    _Round([(int(r.integers(0, 300)), int(r.integers(0, 20))) for _ in range(150)], 8, 2, 8, 8, seed=6).check()


@pytest.mark.parametrize("hq,hkv,requests", [(8, 2, 40), (64, 4, 5), (64, 4, 33), (6, 6, 70), (16, 1, 2)])
def test_attention_of_trees_of_all_sizes_side_by_side(hq, hkv, requests):
    """Trees of one tile's rows, of more, of many items and of none, behind contexts of no token to many: shares of the multiprocessors begin and end anywhere."""
    r = np.random.default_rng(requests)
    counts = [1, 64, 0, 33, 8, 17, 2, 40]
    _Round([(int(r.integers(0, 4) and r.integers(0, 700)), counts[i % 8]) for i in range(requests)], hq, hkv, 8, 6, seed=requests).check()


def test_attention_of_a_long_context_beside_short_ones():
    _Round([(9000, 30), (3, 1), (700, 64), (0, 2)], 16, 2, 4, 8, seed=7).check()


@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 6)])
def test_masks_of_any_kind(kb, vb):
    """Masks that name what a tree does not have, nodes that do not see themselves, rows that see nothing."""
    def masks(c, words, r):
        m = r.integers(0, 1 << 32, (c, words), dtype=np.uint64).astype(np.uint32)          # bits behind the last node too
        m[::3] = 0
        return m
    rd = _Round([(0, 40), (5, 70), (0, 1), (80, 7)], 4, 2, kb, vb, seed=8, masks=masks, words=4)
    got = rd.check()
    empty = ~(rd.sees[:40, 0].astype(bool) | (rd.sees[:40, 1] & 255).astype(bool))
    assert empty.any() and (got[:40][torch.from_numpy(empty).to(DEV)] == 0).all()


def test_rows_of_no_request_and_neighbours_in_wider_rows_stay():
    rd = _Round([(30, 5), (64, 3)], 4, 2, 8, 8, seed=9)
    wide_q, wide = torch.full((14, 4 * D + 32), 3.0, device=DEV, dtype=torch.bfloat16), torch.full((14, 4 * D + 16), 7.0, device=DEV, dtype=torch.bfloat16)
    wide_q[2:10, 8:8 + 4 * D] = rd.q
    cache, table, slots, row0, *rest = rd.args()
    masks = torch.full((14, 3), -1, dtype=I32, device=DEV)
    masks[2:10, 1:2] = rest[2]
    wide_table = torch.full((table.shape[0], table.shape[1] + 3), -5, dtype=I32, device=DEV)
    wide_table[:, :table.shape[1]] = table
    out = K.tree_attention(wide_q[:, 8:8 + 4 * D], wide[:, 8:8 + 4 * D], cache, wide_table[:, :table.shape[1]], slots, row0 + 2, *rest[:2], masks[:, 1:2], *rest[3:])
    assert torch.equal(out[2:10], rd.run())
    assert (wide[:2] == 7).all() and (wide[10:] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 8 + 4 * D:] == 7).all()


def test_requests_that_are_told_wrongly_are_zeros_and_said():
    rd = _Round([(30, 5), (64, 3), (20, 40)], 4, 2, 8, 8, seed=10)
    want = rd.run()
    for change in (("request", 0, 99), ("request", 0, -1), ("start", 0, 9999), ("start", 0, -1), ("masks", None, None)):
        cache, table, slots, row0, count, start, masks, *rest = rd.args()
        if change[0] == "request":
            slots[change[1]] = change[2]
        elif change[0] == "start":
            start[change[1]] = change[2]
        else:
            masks = masks[:, :1].contiguous()
        out, ws = torch.full_like(rd.q, 7.0), K.Workspace(torch.device(DEV, 0), 16, 16, 16)
        K.tree_attention(rd.q, out, cache, table, slots, row0, count, start, masks, *rest, ws=ws)
        with pytest.raises(NativeLibraryError):
            ws.check_status()
        hit = slice(8, 48) if masks.shape[1] == 1 else slice(0, 5)
        assert (out[hit] == 0).all()
        out[hit] = want[hit]
        assert torch.equal(out, want)
    for what in (("count", 0, 99), ("count", 0, -3), ("row0", 0, -2), ("row0", 0, 47)):
        cache, table, slots, row0, count, start, *rest = rd.args()
        (count if what[0] == "count" else row0)[what[1]] = what[2]
        out, ws = torch.full_like(rd.q, 7.0), K.Workspace(torch.device(DEV, 0), 16, 16, 16)
        K.tree_attention(rd.q, out, cache, table, slots, row0, count, start, *rest, ws=ws)
        with pytest.raises(NativeLibraryError):
            ws.check_status()
        assert (out[:5] == 7).all() and torch.equal(out[5:], want[5:])


def test_pages_that_are_not_there_are_said():
    rd = _Round([(100, 5), (64, 3)], 4, 2, 8, 8, seed=11)
    want = rd.run()
    for page in (-1, 1 << 30, rd.cache.shape[0]):
        table = rd.table.clone()
        table[int(rd.slots[0]), 2] = page
        cache, _, *rest = rd.args()
        out, ws = torch.full_like(rd.q, 7.0), K.Workspace(torch.device(DEV, 0), 16, 16, 16)
        K.tree_attention(rd.q, out, cache, table, *rest, ws=ws)
        with pytest.raises(NativeLibraryError):
            ws.check_status()
        assert torch.equal(out[5:], want[5:])


@pytest.mark.parametrize("kb,vb", [(8, 8), (6, 4)])
@pytest.mark.parametrize("which,bad", [(0, float("nan")), (1, float("nan")), (1, float("inf")), (0, float("inf"))])
def test_values_that_are_not_finite_reach_those_who_see_them(kb, vb, which, bad):
    """In the context, and at a node that some rows do not see."""
    rd = _Round([(70, 12), (40, 12)], 4, 1, kb, vb, seed=12)
    want = rd.run()
    scales = rd.scales()[which]
    for req, tok in ((0, 33), (1, 40 + 5)):
        page = int(rd.table[int(rd.slots[req]), tok // 16])
        old = scales[page, :, tok % 16].clone()
        scales[page, :, tok % 16] = bad
        out = rd.run()
        scales[page, :, tok % 16] = old
        node = tok - rd.sizes[req][0]
        rows = np.arange(24) // 12 == req
        if node >= 0:
            rows &= (rd.sees[:, 0] >> np.uint32(node) & 1).astype(bool)
        hit = torch.from_numpy(rows).to(DEV)
        assert not torch.isfinite(out[hit].float()).all(-1).any() and torch.isfinite(out[~hit].float()).all()
        off = (out[~hit].float() - want[~hit].float()).abs()
        assert bool((off <= 2.0 ** -6 * want[~hit].float().abs() + 2.0 ** -7 * want.float().square().mean().sqrt()).all())
        assert torch.equal(out[12 * (1 - req):12 * (2 - req)], want[12 * (1 - req):12 * (2 - req)])


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("low,high", [(0, 9), (0, 13), (13, 0), (0, 25), (25, 0), (-60, -50), (50, 60), (0, -40)])
def test_scales_of_any_size(which, low, high):
    """Scales that grow or shrink from page to page, and rows whose result hangs on the smallest of them: nodes whose queries point along their own keys."""
    rd = _Round([(200, 8)], 4, 1, 8, 8, seed=13)
    n = 208
    s = rd.scales()[which]
    for i in range(13):
        page = int(rd.table[int(rd.slots[0]), i])
        s[page] = (s[page].double() * 2.0 ** round(low + (high - low) * i / 12)).float()
    if which == 1:                                         # (keys as they are: every probability matters)
        rd.check()
        pages = [eager.decode_cache_page(rd.cache[p, 0].cpu(), D, 8, 8) for p in rd.table[int(rd.slots[0]), :13].tolist()]
        k = torch.cat([p[0] for p in pages])[n - 8:n].double()
        sharp = k / k.norm(dim=-1, keepdim=True) * 60
        rd.q = sharp[:, None].expand(8, 4, D).reshape(8, 4 * D).to(DEV).bfloat16()
        rd.sees[:] = np.uint32(1) << np.arange(8, dtype=np.uint32)[:, None]
        rd.check()
    else:
        rd.q = (rd.q.double() * 2.0 ** -max(low, high)).bfloat16()                           # scores of ordinary size at the largest keys
        rd.check()


@pytest.mark.parametrize("up", [-100, -20, 20, 60, 100])
def test_queries_of_any_size(up):
    """The softmax' scale brings the scores back."""
    rd = _Round([(90, 8)], 4, 2, 8, 8, seed=14)
    want = rd.run()
    rd.q = (rd.q.double() * 2.0 ** up).bfloat16()
    assert torch.equal(rd.run(scale=D ** -0.5 * 2.0 ** -up), want)


def test_queries_that_are_not_finite_keep_to_their_rows():
    rd = _Round([(90, 8)], 4, 2, 8, 8, seed=15)
    want = rd.run()
    rd.q[3, 5], rd.q[6, 200] = float("nan"), float("inf")
    got = rd.run()
    assert got[3, :D].isnan().all() and not torch.isfinite(got[6, D:2 * D].float()).any()
    got[3, :D], got[6, D:2 * D] = want[3, :D], want[6, D:2 * D]
    assert torch.equal(got, want)


def test_attention_on_a_stream_and_in_a_graph():
    """The same bits eagerly, on another stream, captured and replayed, with the lengths changed between replays."""
    rd = _Round([(300, 20), (64, 3), (7, 64)], 32, 4, 8, 8, seed=16)
    want = rd.run()
    assert torch.equal(rd.run(), want)
    args, out, ws = rd.args(), torch.zeros_like(rd.q), K.Workspace(torch.device(DEV, 0), 16, 16, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.tree_attention(rd.q, out, *args, ws=ws)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        K.tree_attention(rd.q, out, *args, ws=ws)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    args[5][0], args[4][2] = 100, 30                       # another context, fewer nodes
    g.replay()
    other = torch.full_like(out, 7.0)
    K.tree_attention(rd.q, other, *args, ws=K.Workspace(torch.device(DEV, 0), 16, 16, 16))
    assert torch.equal(out[:53], other[:53]) and (other[53:] == 7).all() and torch.equal(out[53:], want[53:])
    ws.check_status()


@pytest.mark.parametrize("requests", [1, 90])
@pytest.mark.parametrize("which,low,high", [(0, 0, 25), (1, 0, 25), (1, 25, 0), (0, 0, -40)])
def test_scales_far_apart_of_items_of_both_tiles(requests, which, low, high):
    """129 to 256 rows an item, in parts (one request) and whole: the program in 32 bits, each tile its own rows."""
    rd = _Round([(200 - i % 3, (64, 40, 33)[i % 3]) for i in range(requests)], 4, 2, 8, 8, seed=22)
    s = rd.scales()[which]
    for i, (start, count) in enumerate(rd.sizes):
        held = -(-(start + count) // 16)
        for j in range(held):
            page = int(rd.table[int(rd.slots[i]), j])
            s[page] = (s[page].double() * 2.0 ** round(low + (high - low) * j / (held - 1))).float()
    if which == 0:
        rd.q = (rd.q.double() * 2.0 ** -max(low, high)).bfloat16()
    rd.check()


@pytest.mark.parametrize("which,bad", [(0, float("nan")), (1, float("nan")), (1, float("inf"))])
def test_values_that_are_not_finite_in_items_of_both_tiles(which, bad):
    """At a token of one context and at a node of another tree: 256 rows an item, whole ones and parts."""
    rd = _Round([(70, 64)] * 70 + [(500, 64)], 4, 2, 8, 8, seed=23)
    want = rd.run()
    for req, tok in ((3, 33), (68, 70 + 5), (70, 100)):
        scales = rd.scales()[which]
        page = int(rd.table[int(rd.slots[req]), tok // 16])
        old = scales[page, :, tok % 16].clone()
        scales[page, :, tok % 16] = bad
        out = rd.run()
        scales[page, :, tok % 16] = old
        node = tok - rd.sizes[req][0]
        rows = np.arange(out.shape[0]) // 64 == req
        if node >= 0:
            rows &= (rd.sees[:, node >> 5] >> np.uint32(node & 31) & 1).astype(bool)
        hit, others = torch.from_numpy(rows).to(DEV), torch.from_numpy(np.arange(out.shape[0]) // 64 != req).to(DEV)
        assert rows.any() and not torch.isfinite(out[hit].float()).all(-1).any() and torch.isfinite(out[~hit].float()).all()
        assert torch.equal(out[others], want[others])
        # rows of the tree that do not see it: the same in 32 bits
        ref, tol = rd.truth()
        off = (out.cpu().double() - ref).abs()
        assert bool((off <= tol + 1e-30)[~torch.from_numpy(rows)].all())


def test_values_far_apart_behind_a_long_context():
    """A context of 160000 tokens whose scales take the program in 32 bits: all rows of an item of 256 by one CTA.

    The context is the same 256 tokens over and over, so that each counts as often as it is there.  n products are summed in 32 bits, one after the other: each addition is
    off by 2^-24 of what is there at most, in the sum and in the output.  A score is off by 2^-24 of the sum of its products' magnitudes for each of 16 roundings
    at most, exponentials by 2^-20, the result by 2^-8."""
    times, sms = 625, K.sm_count(torch.device(DEV, 0))
    rd = _Round([(256, 64)], 4, 1, 8, 8, seed=21)
    rd.scales()[1][int(rd.table[int(rd.slots[0]), 3])] *= 2.0 ** -24
    ids = rd.table[int(rd.slots[0]), :20]
    table = torch.cat([ids[:16].repeat(times), ids[16:]])[None].contiguous()
    cache, _, _, _, _, _, masks, *rest = rd.args()
    out, ws = torch.full((64 * sms, 4 * D), 7.0, device=DEV, dtype=torch.bfloat16), K.Workspace(torch.device(DEV, 0), 16, 16, 16)
    K.tree_attention(rd.q.repeat(sms, 1), out, cache, table, _i32([0] * sms), _i32(np.arange(sms) * 64), _i32([64] * sms), _i32([256 * times] * sms), masks.repeat(sms, 1), *rest, ws=ws)
    ws.check_status()
    pages = [eager.decode_cache_page(rd.cache[p, 0].cpu(), D, 8, 8) for p in ids.tolist()]
    k, v = (torch.cat([page[x] for page in pages]).double() for x in (0, 1))
    q, n = rd.q.cpu().double().view(64, 4, D), 256 * times + 64
    z = torch.einsum("cgd,td->cgt", q, k) * D ** -0.5
    off = (torch.einsum("cgd,td->cgt", q.abs(), k.abs()) * D ** -0.5 * 16 * 2.0 ** -24).amax(-1, keepdim=True)
    often = torch.full((64, 1, 320), float(times), dtype=torch.float64)
    often[:, 0, 256:] = torch.from_numpy(((rd.sees[:, :, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(64, -1).astype(np.float64))
    p = often * torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    ref, tol = torch.einsum("cgt,td->cgd", p, v), (torch.expm1(2 * off) + 2 * n * 2.0 ** -24 + 2.0 ** -19) * torch.einsum("cgt,td->cgd", p, v.abs())
    assert bool(((out[:64].cpu().double() - ref.reshape(64, -1)).abs() <= (tol + 2.0 ** -8 * ref.abs()).reshape(64, -1)).all())
    assert torch.equal(out, out[:64].repeat(sms, 1))


def test_no_requests():
    rd = _Round([(30, 5)], 4, 2, 8, 8, seed=17)
    cache, table, slots, row0, count, start, *rest = rd.args()
    out = torch.full_like(rd.q, 7.0)
    K.tree_attention(rd.q, out, cache, table, slots[:0], row0[:0], count[:0], start[:0], *rest)
    K.tree_attention(rd.q, out, cache, table, slots, row0, count * 0, start, *rest)
    assert (out == 7).all()
    K.workspace(torch.device(DEV, 0)).check_status()


# ------------------------------------------------------------------------------------------------- logits
def _adjusted(x, request, history, length, prompt, rep, freq, pres, bias, mask, drafts):
    """Plain loops in 64 bits; rounds where the definition says."""
    x = x.copy()
    rows, vocab = x.shape
    for r in range(rows):
        q = request[r] if request is not None else r
        if 0 <= q < len(length):
            said = [int(t) for t in history[q, :length[q]]]
            new = said[prompt[q] if prompt is not None else 0:]
            if drafts is not None:
                tokens, sees, row0 = drafts
                more = [int(tokens[row0[q] + j]) for j in range(1, 32 * sees.shape[1]) if sees[r, j // 32] >> np.uint32(j % 32) & 1 and 0 <= row0[q] and row0[q] + j < rows]
                said, new = said + more, new + more
            for t in set(said):
                if 0 <= t < vocab and rep is not None:
                    x[r, t] = x[r, t] / rep[q] if x[r, t] > 0 else x[r, t] * rep[q]
            for t in set(new):
                if 0 <= t < vocab:
                    x[r, t] -= new.count(t) * (freq[q] if freq is not None else 0.0)
                    x[r, t] -= pres[q] if pres is not None else 0.0
            if bias is not None:
                at, ids, values = bias
                for t, v in {int(t): v for t, v in zip(ids[at[q]:at[q + 1]], values[at[q]:at[q + 1]])}.items():
                    if 0 <= t < vocab:
                        x[r, t] += v
        if mask is not None:
            allowed = (mask[r % len(mask)][np.arange(vocab) >> 5] >> (np.arange(vocab) & 31).astype(np.uint32)) & 1
            x[r, allowed == 0] = -np.inf
    return x


class _Wishes:
    def __init__(self, rows, vocab, n, most, f32=False, seed=0, nodes=0, bias=0, masked=False, request=True, full=True, pitch=0, odd=0):
        r = np.random.default_rng(seed)
        dt = torch.float32 if f32 else torch.bfloat16
        flat = torch.zeros(rows * (vocab + pitch) + odd + 64, dtype=dt, device=DEV)
        self.logits = flat[odd:odd + rows * (vocab + pitch)].view(rows, vocab + pitch)[:, :vocab]
        self.logits.copy_(torch.from_numpy(r.standard_normal((rows, vocab)) * 4))
        h = {"history": (vocab * r.random((n, most)) ** 3).astype(int), "length": r.integers(0, most + 1, n), "request": r.integers(-1, n, rows) if request else None}
        h["history"][:, ::7] = r.integers(-3, vocab + 3, h["history"][:, ::7].shape)
        h["prompt"] = (h["length"] * r.random(n)).astype(int) if full else None
        f = lambda lo, hi: r.uniform(lo, hi, n).astype(np.float32) if full else None         # noqa: E731
        h["rep"], h["freq"], h["pres"] = r.uniform(0.7, 1.6, n).astype(np.float32), f(-1, 1), f(-1, 1)
        h["bias"] = h["mask"] = h["drafts"] = None
        if bias:
            at = np.concatenate([[0], r.integers(0, bias + 1, n).cumsum()])
            h["bias"] = (at, r.integers(-2, vocab + 2, at[-1]), r.uniform(-9, 9, at[-1]).astype(np.float32))      # some twice
        if masked:
            h["mask"] = r.integers(0, 1 << 32, (rows, -(-vocab // 32)), dtype=np.uint64).astype(np.uint32)
        if nodes:
            assert rows == n * nodes
            h["request"] = np.repeat(np.arange(n), nodes)
            h["drafts"] = ((vocab * r.random(rows) ** 3).astype(int), np.concatenate([tree_masks(_parents(nodes, r), -(-nodes // 32) + 1) for _ in range(n)]), np.arange(n) * nodes)
        self.h = h
        d = {k: None if v is None else torch.from_numpy(v).to(DEV) if v.dtype == np.float32 else _i32(v) for k, v in h.items() if not isinstance(v, tuple) and k != "mask"}
        u = lambda a: torch.from_numpy(a.view(np.int32)).to(DEV)                              # noqa: E731
        self.kw = dict(request=d["request"], history=d["history"], length=d["length"], prompt=d["prompt"], repetition=d["rep"], frequency=d["freq"], presence=d["pres"],
                       bias=None if h["bias"] is None else (_i32(h["bias"][0]), _i32(h["bias"][1]), torch.from_numpy(h["bias"][2]).to(DEV)),
                       mask=None if h["mask"] is None else u(h["mask"]), drafts=None if h["drafts"] is None else (_i32(h["drafts"][0]), u(h["drafts"][1]), _i32(h["drafts"][2])))
        self.eps = 2.0 ** -24 if f32 else 2.0 ** -8

    def check(self, out=None):
        """fp32 steps (at most four, each off by 2^-24 of what it gives or takes) and one rounding to the logits' type."""
        x = self.logits.double().cpu().numpy()
        ref = _adjusted(x, **self.h)
        flat = self.logits._base
        around = flat.clone()
        got = K.adjust_logits(self.logits, out=out, **self.kw).double().cpu().numpy()
        if out is None:
            inside = torch.zeros_like(flat, dtype=torch.bool).as_strided(self.logits.shape, self.logits.stride(), self.logits.storage_offset())
            inside.fill_(True)
            assert torch.equal(flat[~inside._base], around[~inside._base])
        f = lambda a: 0.0 if self.h[a] is None else np.abs(self.h[a]).max()                  # noqa: E731
        sizes = np.abs(x) * 2 + np.abs(np.where(np.isfinite(ref), ref, 0)) + 20
        same = np.isinf(ref)
        assert np.array_equal(np.isneginf(got), same)
        with np.errstate(invalid="ignore"):
            off, tol = np.abs(got - ref), self.eps * np.abs(ref) + 5 * 2.0 ** -24 * (sizes + self._counted(f("freq")))
        assert bool((same | (off <= tol)).all()), np.nanmax(np.where(same, 0, off / tol))
        untouched = ref == x
        assert np.array_equal(got[untouched], x[untouched])

    def _counted(self, freq):
        return freq * (self.h["history"].shape[1] + 64)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,vocab,n,most", [(1, 1000, 1, 50), (5, 33, 3, 40), (3, 1, 2, 9), (9, 50257, 4, 3000), (2, 151936, 2, 700), (40, 8192, 40, 1), (3, 8193, 3, 2000), (2, 100, 2, 0), (300, 9000, 50, 60)])
def test_logits_as_requests_want_them(rows, vocab, n, most, f32):
    _Wishes(rows, vocab, n, most, f32, seed=rows + vocab, bias=30, masked=True).check()
    _Wishes(rows, vocab, n, most, f32, seed=rows + vocab + 1, bias=5).check()
    _Wishes(rows, vocab, n, most, f32, seed=rows + vocab + 2).check(torch.zeros(rows, vocab, dtype=torch.float32 if f32 else torch.bfloat16, device=DEV))
    _Wishes(rows, vocab, max(n, rows), most, f32, seed=rows + vocab + 3, request=False, full=False).check()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("pitch,odd", [(0, 1), (3, 0), (8, 0), (5, 3), (16, 4)])
def test_logits_of_any_alignment(pitch, odd, f32):
    _Wishes(6, 5000, 4, 300, f32, seed=pitch + odd, bias=9, masked=True, pitch=pitch, odd=odd).check()
    w = _Wishes(6, 5000, 4, 300, f32, seed=pitch + odd, bias=9, pitch=pitch, odd=odd)
    w.check(torch.zeros(6, 5003, dtype=w.logits.dtype, device=DEV)[:, :5000])
    w = _Wishes(6, 5000, 4, 300, f32, seed=pitch + odd, bias=9, masked=True, pitch=pitch, odd=odd)
    w.check(torch.zeros(6 * 5000 + 5, dtype=w.logits.dtype, device=DEV)[5:].view(6, 5000))


@pytest.mark.parametrize("n,nodes", [(1, 2), (3, 26), (2, 64), (1, 200)])
def test_logits_of_trees_count_what_leads_to_a_node(n, nodes):
    _Wishes(n * nodes, 3001, n, 100, True, seed=nodes, nodes=nodes, bias=7).check()
    _Wishes(n * nodes, 40, n, 30, False, seed=nodes, nodes=nodes).check()


def test_one_mask_for_all_rows_and_long_lists_of_biases():
    w = _Wishes(4, 9000, 2, 100, True, seed=3, bias=6000)                                    # more entries than a word of the table can name
    w.h["mask"] = np.random.default_rng(1).integers(0, 1 << 32, (1, 282), dtype=np.uint64).astype(np.uint32)
    w.kw["mask"] = torch.from_numpy(w.h["mask"].view(np.int32)).to(DEV).expand(4, 282)
    w.check()


@pytest.mark.parametrize("request_of_row,finite", [(-1, 3.0), (0, 0.75)])
def test_logits_that_are_not_finite(request_of_row, finite):
    w = _Wishes(1, 300, 1, 0, True, seed=4)
    w.logits[0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3.0])
    w.kw.update(request=_i32([request_of_row]), history=_i32(np.arange(4)[None]), length=_i32([4]), prompt=_i32([2]), repetition=torch.full((1,), 2.0, device=DEV), frequency=torch.full((1,), 0.5, device=DEV),
                presence=torch.full((1,), 0.25, device=DEV))
    got = K.adjust_logits(w.logits, **w.kw)[0, :4].tolist()
    assert got[0] != got[0] and got[1:] == [float("inf"), -float("inf"), finite]


def test_adjusting_in_a_graph():
    w = _Wishes(30, 20011, 8, 900, seed=5, bias=20, masked=True)
    out = torch.empty(30, 20011, dtype=torch.bfloat16, device=DEV)
    want = K.adjust_logits(w.logits, out=out, **w.kw).clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.adjust_logits(w.logits, out=out, **w.kw)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------- the round's end
def _walk(target, tokens, parents, depth):
    path, emitted = [0], [target[0]]
    while len(path) < depth:
        nxt = next((j for j in range(path[-1] + 1, len(tokens)) if parents[j] == path[-1] and tokens[j] == emitted[-1]), None)
        if nxt is None:
            break
        path.append(nxt)
        emitted.append(target[nxt])
    return path, emitted


@pytest.mark.parametrize("sizes,depth", [([1], 1), ([8], 5), ([26] * 64, 9), ([1, 0, 256, 33, 64, 2], 40), ([70], 2), ([5] * 300, 5)])
def test_path_that_the_target_agrees_with(sizes, depth):
    r = np.random.default_rng(len(sizes) + depth)
    row0 = np.concatenate([[0], np.cumsum(sizes)])[:-1].astype(int)
    rows = sum(sizes)
    parents = np.concatenate([np.array(_parents(c, r, 3)) for c in sizes if c])
    tokens, target = r.integers(0, 3, rows), r.integers(0, 3, rows)                          # few tokens: siblings alike
    n = len(sizes)
    acc, path, emitted = (torch.full(s, -9, dtype=I32, device=DEV) for s in ((n + 1,), (n + 1, depth), (n + 1, depth)))
    K.verify_tree(_i32(target), _i32(tokens), _i32(parents), _i32(row0), _i32(sizes), acc, path, emitted)
    for i, c in enumerate(sizes):
        s = slice(row0[i], row0[i] + c)
        want = _walk(target[s].tolist(), tokens[s].tolist(), parents[s].tolist(), depth) if c else ([], [])
        pad = [-1] * (depth - len(want[0]))
        assert acc[i].item() == max(len(want[0]) - 1, 0) and path[i].tolist() == want[0] + pad and emitted[i].tolist() == want[1] + pad
    assert acc[n] == -9 and (path[n] == -9).all() and (emitted[n] == -9).all()


def _keep_case(n, start, hkv, kb, vb, paths, layers=3, seed=0):
    r = np.random.default_rng(seed)
    lay = eager.blob_layout(D, kb, vb)
    held = -(-(start + 64) // 16)
    table = r.permutation(n * held + 1)[:n * held].reshape(n, held)
    caches = [torch.from_numpy(r.integers(0, 255, (n * held + 1, hkv, lay["bytes"]), dtype=np.uint8)).to(DEV) for _ in range(layers)]
    for c in caches:
        for a, b in (("k_scale", "v_code"), ("v_scale", "bytes")):
            c[:, :, lay[a]:lay[b]].view(torch.float32).uniform_(0.5, 2.0)
    depth = max(len(p) for p in paths) + 1
    path = np.full((n, depth), -1)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    return caches, table, path, np.array([len(p) - 1 for p in paths])


@pytest.mark.parametrize("kb,vb", BITS)
@pytest.mark.parametrize("start", [0, 5, 16, 43])
def test_kept_tokens_move_up(kb, vb, start):
    """Overlapping and far moves within and across pages; every other bit of the cache stays."""
    paths = [[0], [0, 1, 2], [0, 2, 3, 4, 5, 6, 7, 8, 9, 10], [0, 17, 33, 49], [0, 1, 5, 20, 21, 22, 63], [0, 63]]
    n, hkv = len(paths), 2
    caches, table, path, accepted = _keep_case(n, start, hkv, kb, vb, paths, seed=kb + vb + start)
    want = [c.cpu().clone() for c in caches]
    before = [c.cpu().clone() for c in caches]
    K.keep_tokens(K.LayerCaches(caches, hkv, D, kb, vb), _i32(table), _i32(np.arange(n)), _i32(np.full(n, start)), _i32(accepted), _i32(path))
    K.workspace(torch.device(DEV, 0)).check_status()
    for c, old in zip(caches, before):
        c = c.cpu()
        for i, p in enumerate(paths):
            for h in range(hkv):
                new_k, new_v = zip(*(eager.decode_cache_page(c[pg, h], D, kb, vb) for pg in table[i].tolist()))
                old_k, old_v = zip(*(eager.decode_cache_page(old[pg, h], D, kb, vb) for pg in table[i].tolist()))
                for new, was in ((torch.cat(new_k), torch.cat(old_k)), (torch.cat(new_v), torch.cat(old_v))):
                    ref = was.clone()
                    for k, node in enumerate(p):
                        ref[start + k] = was[start + node]
                    assert torch.equal(new, ref)
        spare = sorted(set(range(len(c))) - set(table.reshape(-1).tolist()))
        assert torch.equal(c[spare], old[spare])
    assert len(want) == 3


def test_paths_that_do_not_rise_and_pages_that_are_not_there_move_nothing_and_are_said():
    paths = [[0, 3, 2], [0, 5], [0, 7]]
    caches, table, path, accepted = _keep_case(3, 10, 2, 8, 8, paths, seed=3)
    table[1, 0] = 1 << 20
    for hit in (dict(), dict(request=[0, 1, 99]), dict(start=[10, 10, -4]), dict(accepted=[2, 1, 9])):
        now = [c.clone() for c in caches]
        ws = K.Workspace(torch.device(DEV, 0), 16, 16, 16)
        acc = np.array(hit.get("accepted", accepted))
        if not hit:
            acc[2] = 0
        path0 = path.copy()
        path0[0, 1] = 0                                    # does not rise at once
        K.keep_tokens(K.LayerCaches(now, 2, D, 8, 8), _i32(table), _i32(hit.get("request", [0, 1, 2])), _i32(hit.get("start", [10] * 3)), _i32(acc), _i32(path0), ws=ws)
        with pytest.raises(NativeLibraryError):
            ws.check_status()
        assert all(torch.equal(a, b) for a, b in zip(now, caches))


@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 6), (6, 4)])
def test_kept_paths_longer_than_a_warp(kb, vb):
    """32, 33 and 64 places, some of whose lines move and some stay, beside a short one."""
    paths = [list(range(30)) + [33, 40, 63], list(range(20)) + list(range(21, 35)), [0] + list(range(30, 62)), [0] + list(range(1, 64)), [0, 2]]
    n, hkv, start = len(paths), 2, 13
    caches, table, path, accepted = _keep_case(n, start, hkv, kb, vb, paths, layers=2, seed=30 + kb)
    before = [c.cpu().clone() for c in caches]
    K.keep_tokens(K.LayerCaches(caches, hkv, D, kb, vb), _i32(table), _i32(np.arange(n)), _i32(np.full(n, start)), _i32(accepted), _i32(path))
    K.workspace(torch.device(DEV, 0)).check_status()
    for c, old in zip(caches, before):
        for i, p in enumerate(paths):
            for h in range(hkv):
                new, was = ([torch.cat(x) for x in zip(*(eager.decode_cache_page(t[pg, h], D, kb, vb) for pg in table[i].tolist()))] for t in (c.cpu(), old))
                for a, b in zip(new, was):
                    ref = b.clone()
                    ref[start:start + len(p)] = b[[start + node for node in p]]
                    assert torch.equal(a, ref)


@pytest.mark.parametrize("path,page", [([0, 3, 2], None), ([0, 2, 4, 6, 8, 8, 9], None), ([0, 2, 4, 6, 8, 9, -1], None), (list(range(0, 70, 2)) + [60], None),
                                       ([0, 3, 20], 1), ([0, 3, 4, 9, 20, 21], 1), ([0, 3, 4, 5, 6, 7, 8, 9, 40], 3)])
def test_paths_that_are_wrong_further_on_move_nothing(path, page):
    """Lines of a path before the place where it is wrong stay, and other requests' move."""
    paths = [path, [0, 3, 5]]
    caches, table, want_path, accepted = _keep_case(2, 10, 2, 8, 8, paths, seed=4)
    if page is not None:
        table[0, page] = -1
    now, only = ([c.clone() for c in caches] for _ in range(2))
    ws = K.Workspace(torch.device(DEV, 0), 16, 16, 16)
    K.keep_tokens(K.LayerCaches(now, 2, D, 8, 8), _i32(table), _i32([0, 1]), _i32([10] * 2), _i32(accepted), _i32(want_path), ws=ws)
    with pytest.raises(NativeLibraryError):
        ws.check_status()
    K.keep_tokens(K.LayerCaches(only, 2, D, 8, 8), _i32(table), _i32([1]), _i32([10]), _i32(accepted[1:]), _i32(want_path[1:]), ws=ws)
    ws.check_status()
    assert all(torch.equal(a, b) for a, b in zip(now, only)) and not all(torch.equal(a, b) for a, b in zip(now, caches))


# ------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kb,vb", [(8, 8), (4, 8), (6, 6)])
def test_a_round_leaves_the_cache_of_a_chain(kb, vb):
    """Attention over a tree, its greedy walk and the move: what the next round reads is what decoding the accepted tokens one by one has."""
    r = np.random.default_rng(kb)
    hkv, hq, start, nodes = 2, 8, 37, 20
    lay = eager.blob_layout(D, kb, vb)
    pages = -(-(start + nodes) // 16)
    inv = torch.from_numpy((10000.0 ** (-np.arange(0, 64) / 64)).astype(np.float32)).to(DEV)
    table = _i32(r.permutation(pages)[None])

    def write(cache, values, positions, slots):
        q = torch.empty(len(positions), hq * D, dtype=torch.bfloat16, device=DEV)
        at = [int(table[0, s // 16]) * 16 + s % 16 for s in slots]
        K.rope_kv_write(values, q, cache, _i32(positions), _i32(at), inv, hq, hkv, D, kb, vb)
        return q

    vals = torch.from_numpy(r.standard_normal((start + nodes, (hq + 2 * hkv) * D)).astype(np.float32)).to(DEV).bfloat16()
    tree, chain = (torch.zeros(pages, hkv, lay["bytes"], dtype=torch.uint8, device=DEV) for _ in range(2))
    parents = _parents(nodes, r, 5)
    depth = np.zeros(nodes, dtype=int)
    for j in range(1, nodes):
        depth[j] = depth[parents[j]] + 1
    tokens = r.permutation(nodes)
    deepest = int(depth.argmax())
    way = [deepest]
    while way[0]:
        way.insert(0, parents[way[0]])
    target = np.full(nodes, 999)
    for a, b in zip(way, way[1:]):
        target[a] = tokens[b]
    for c in (tree, chain):
        write(c, vals[:start], np.arange(start), np.arange(start))
    q = write(tree, vals[start:], start + depth, start + np.arange(nodes))
    out = torch.empty_like(q)
    one = _i32([0])
    K.tree_attention(q, out, tree, table, one, one, _i32([nodes]), _i32([start]), torch.from_numpy(tree_masks(parents).view(np.int32)).to(DEV), hq, hkv, D, kb, vb)
    acc, path, emitted = torch.zeros(1, dtype=I32, device=DEV), torch.zeros(1, nodes, dtype=I32, device=DEV), torch.zeros(1, nodes, dtype=I32, device=DEV)
    K.verify_tree(_i32(target), _i32(tokens), _i32(parents), one, _i32([nodes]), acc, path, emitted)
    assert path[0, :len(way)].tolist() == way and acc.item() == len(way) - 1
    K.keep_tokens(K.LayerCaches([tree], hkv, D, kb, vb), table, one, _i32([start]), acc, path)
    for k, node in enumerate(way):
        x = vals[start + node:start + node + 1]
        qc = write(chain, x, [start + k], [start + k])
        oc = torch.empty(1, hq, D, dtype=torch.bfloat16, device=DEV)
        K.paged_attention(qc.view(1, hq, D), oc, chain, table, one, one, _i32([1]), _i32([start + k + 1]), hq, hkv, D, kb, vb)
        a, b = out[node].float(), oc.view(-1).float()
        assert ((a - b).abs() <= 2.0 ** -6 * b.abs() + 2.0 ** -7 * b.square().mean().sqrt()).all()
    for h in range(hkv):
        for j, page in enumerate(table[0].tolist()):
            for x, y in zip(eager.decode_cache_page(tree[page, h].cpu(), D, kb, vb), eager.decode_cache_page(chain[page, h].cpu(), D, kb, vb)):
                m = max(0, min(16, start + len(way) - 16 * j))
                assert torch.equal(x[:m], y[:m])
    K.workspace(torch.device(DEV, 0)).check_status()
