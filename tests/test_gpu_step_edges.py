"""Edges of the operators around a step's shared layers."""
import math
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from cubic_serve_b200.ops import kernels as K
from test_gpu_step_operators import _adapter_case, _adapter_truth, _check_adapter

pytestmark = pytest.mark.gpu
DEV = "cuda"
I32 = torch.int32
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


# ------------------------------------------------------------------------------------------------- adapters
@pytest.mark.parametrize("rows", [1, 40, 700])
@pytest.mark.parametrize("rank,widths", [(16, (96, 32, 64)), (40, (64, 64)), (128, (32, 32, 32))])
def test_a_section_without_matrices_is_left_alone(rows, rank, widths):
    """An infinity or NaN in x meets an adapter that has no matrices for a section: that section's columns are y, to the bit."""
    k, S = 264, len(widths)
    x, y, a, b, scale = _adapter_case(rows, 2, rank, k, widths, None, seed=6)
    bank = K.AdapterBank(a, b, scale, widths)
    cut = lambda i: b[0, sum(widths[:i]):sum(widths[:i + 1])]        # noqa: E731
    for none in range(S):
        bank.load(0, [None if i == none else a[0, i * rank:i * rank + rank] for i in range(S)], [None if i == none else cut(i) for i in range(S)], 1.5)
        x2 = x.clone()
        x2[0, 7] = math.inf
        x2[rows // 2, 100] = math.nan
        x2[rows - 1, 263] = -math.inf
        ids = torch.zeros(rows, dtype=I32, device=DEV)
        plan = K.adapter_rows(ids, K.AdapterRows(rows, 2, S * rank, DEV))
        lo = sum(widths[:none])
        for in_place in (False, True):
            got = K.adapter_add(x2, y.clone(), bank, plan) if in_place else K.adapter_add(x2, y, bank, plan, out=torch.empty_like(y))
            assert torch.equal(got[:, lo:lo + widths[none]], y[:, lo:lo + widths[none]])
            rest = torch.cat([got[rows // 2, :lo], got[rows // 2, lo + widths[none]:]])
            assert bool(rest.isnan().all()), "what is not finite reaches the columns of the other sections"


@pytest.mark.parametrize("rows", [33, 600])
def test_sections_of_different_ranks(rows):
    """Ranks 24, none and 3 of one adapter, all of another: the ranks behind a section's own are nobody's, also where x is not finite."""
    widths, rank, k = (64, 32, 40), 24, 136
    x, y, a, b, scale = _adapter_case(rows, 2, rank, k, widths, None, seed=8)
    bank = K.AdapterBank(a, b, scale, widths)
    bank.load(1, [a[1, :24], None, a[1, 48:51]], [b[1, :64], None, b[1, 96:, :3]], float(scale[1]))
    a[1, 24:48], a[1, 51:], b[1, 64:96], b[1, 96:, 3:] = 0, 0, 0, 0
    ids = np.arange(rows) % 3 - 1
    plan = K.adapter_rows(torch.tensor(ids.tolist(), dtype=I32, device=DEV), K.AdapterRows(rows, 2, 72, DEV))
    want, err = _adapter_truth(x, y, a, b, scale, widths, ids)
    got = K.adapter_add(x, y, bank, plan, out=torch.empty_like(y))
    assert bool(((got.double() - want).abs() <= err).all())
    x[2, 5], b[1, 96:, :3] = math.inf, b[1, 96:, :3].abs() + 0.1
    bank.load(1, [a[1, :24], None, a[1, 48:51].abs() + 0.1], [b[1, :64], None, b[1, 96:, :3]], float(scale[1]))
    got = K.adapter_add(x, y, bank, plan, out=torch.empty_like(y))
    assert torch.equal(got[2, 64:96], y[2, 64:96]) and bool((got[2, 96:] == math.inf).all())


@pytest.mark.parametrize("rows", [20, 600])
@pytest.mark.parametrize("rank", [24, 100])
def test_ranks_that_are_not_in_use_reach_nothing(rows, rank):
    """A bank made over buffers with NaN behind the ranks in use, and an empty slot that is NaN throughout."""
    widths, ranks = (64, 32), (rank, 5, 0)
    x, y, a, b, scale = _adapter_case(rows, 3, rank, 136, widths, None, seed=2)
    ids = np.arange(rows) % 4 - 1
    want, err = _adapter_truth(x, y, a, b, scale, widths, ids, ranks)
    for s, r in enumerate(ranks):
        a.view(3, 2, rank, 136)[s, :, r:] = math.nan
        b[s, :, r:] = math.nan
    scale[2] = math.nan
    bank = K.AdapterBank(a, b, scale, widths, ranks=torch.tensor(ranks, dtype=I32, device=DEV))
    plan = K.adapter_rows(torch.tensor(ids.tolist(), dtype=I32, device=DEV), K.AdapterRows(rows, 3, 2 * rank, DEV))
    got = K.adapter_add(x, y, bank, plan, out=torch.empty_like(y))
    assert bool(((got.double() - want).abs() <= err).all()) and torch.equal(got[3::4], y[3::4])


@pytest.mark.parametrize("rows,slots", [(1, 8), (48, 16), (200, 5), (513, 3), (900, 40)])
@pytest.mark.parametrize("rank,widths", [(16, (96, 32)), (64, (64, 32, 32))])
def test_a_row_keeps_its_bits_whatever_its_neighbours_are(rows, slots, rank, widths):
    """As many rows and slots: a row's result is the same bits wherever it stands, whatever the other rows hold and whichever adapters these name."""
    k = 1100 // 8 * 8
    x, y, a, b, scale = _adapter_case(rows, slots, rank, k, widths, None, seed=rows)
    bank, plan = K.AdapterBank(a, b, scale, widths), K.AdapterRows(rows, slots, len(widths) * rank, DEV)
    r = np.random.default_rng(rows)
    mine = x[0].clone(), y[0].clone()
    seen = []
    for trial in range(6):
        at = int(r.integers(0, rows)) if trial else 0
        ids = r.integers(-1, slots, rows).astype(np.int32) if trial % 2 else np.full(rows, slots // 2, dtype=np.int32)
        ids[at] = slots // 2
        x2, y2 = x[torch.from_numpy(r.permutation(rows)).to(DEV)] * (1.0 + trial), y.clone()
        x2[at], y2[at] = mine
        K.adapter_rows(torch.from_numpy(ids).to(DEV), plan)
        seen.append(K.adapter_add(x2, y2, bank, plan, out=torch.empty_like(y) if trial % 3 else None)[at].clone())
    assert all(torch.equal(seen[0], s) for s in seen[1:])


def test_a_row_among_other_numbers_of_rows_is_within_its_bound():
    """The order of the sums follows the numbers of rows and slots: the same row alone and among 47, 511, 512 and 1200 others is within the bound each time."""
    k, rank, widths = 2048, 32, (128, 64)
    for slots in (2, 60):
        x, y, a, b, scale = _adapter_case(1201, slots, rank, k, widths, None, seed=slots)
        bank = K.AdapterBank(a, b, scale, widths)
        want, err = _adapter_truth(x[:1], y[:1], a, b, scale, widths, np.array([1]))
        for rows in (1, 48, 512, 513, 1201):
            ids = torch.arange(1, rows + 1, dtype=I32, device=DEV) % slots
            plan = K.adapter_rows(ids, K.AdapterRows(rows, slots, 2 * rank, DEV))
            got = K.adapter_add(x[:rows], y[:rows], bank, plan, out=torch.empty(rows, 192, device=DEV, dtype=torch.bfloat16))
            assert bool(((got[:1].double() - want).abs() <= err).all())


@pytest.mark.parametrize("rows,slots,rank,k,widths,ranks", [
    (513, 3, 16, 520, (96, 32, 32), None), (640, 5, 32, 264, (64, 64, 64), None), (777, 2, 64, 136, (128, 32, 32), None), (600, 4, 128, 264, (64, 32, 32), None), (1025, 9, 20, 72, (32, 40), None),
    (530, 3, 32, 512, (256,), None), (700, 6, 64, 200, (96, 32), (64, 0, 5, 33, 1, 17)), (640, 4, 128, 136, (96,), (128, 0, 70, 3)), (520, 1, 48, 1032, (64, 64, 32, 32), None),
    (2000, 600, 16, 64, (64, 64), None), (513, 2, 16, 8, (8,), (16, 9)),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_many_rows_of_every_rank_against_64_bits(rows, slots, rank, k, widths, ranks, in_place):
    """More rows than the launch for few takes: three and four sections, every stored rank, ranks in use, strides, in place."""
    ids = np.random.default_rng(rows).integers(-1, slots + 1, rows)
    _check_adapter(rows, slots, rank, k, widths, ids, seed=rows + rank, ranks=ranks, in_place=in_place, pad_x=16, pad_y=24)


def test_many_rows_of_one_adapter_and_of_runs():
    """Runs that end inside a tile of 64 and a strip of sixteen; one adapter for all rows; rows without one in between."""
    rows, slots = 1111, 5
    for ids in (np.full(rows, 2), np.arange(rows) * slots // rows, np.where(np.arange(rows) % 97 < 50, 3, -1), np.arange(rows) % 7 - 1):
        a = _check_adapter(rows, slots, 32, 136, (64, 32, 32), ids, seed=3, in_place=True, pad_y=8)
        assert torch.equal(a, _check_adapter(rows, slots, 32, 136, (64, 32, 32), ids, seed=3, pad_y=8))


# ------------------------------------------------------------------------------------------------- served steps
def _laid_out(**kw):
    from test_gpu_step_serving import _executor
    return _executor(device_layout=True, **kw)


@pytest.mark.parametrize("graphs", [True, False])
def test_a_step_that_the_device_could_not_place_is_an_error(graphs):
    """Pages that go missing between staging and layout: the step's ids are not handed out, and the executor serves on."""
    from cubic_serve_b200.executor.gpu_executor import Segment
    ex = _laid_out(graphs=graphs)
    if graphs:
        ex.capture_decode_graphs([1, 2, 4, 8])
    seg = lambda start, n, sample=True: Segment(0, list(range(1, n + 1)), start, [5, 6, 7], sample, uid=9)        # noqa: E731
    first = ex.execute([seg(0, 30)]).tolist()
    stage = ex.builder.stage_layout
    for s in (seg(30, 1), seg(30, 10), seg(30, 10, False)):                 # a decode step, a portion with a sampled row, one without
        ex.builder.forget_device_rows()
        ex.builder.stage_layout = lambda segs: stage(segs) - 1
        with pytest.raises(RuntimeError, match="not enough pages"):
            ex.execute([s])
        ex.builder.stage_layout = stage
        assert ex.execute([seg(0, 30)]).tolist() == first
    # two steps under way: the error belongs to the one that met it
    a = ex.launch([seg(30, 1)])
    ex.builder.forget_device_rows()
    ex.builder.stage_layout = lambda segs: stage(segs) - 1
    b = ex.launch([seg(31, 1)], feedback_rows=1)
    ex.builder.stage_layout = stage
    assert len(ex.collect(a)) == 1
    with pytest.raises(RuntimeError, match="not enough pages"):
        ex.collect(b)
    assert ex.execute([seg(0, 30)]).tolist() == first


def test_padding_is_poisoned_in_steps_laid_out_on_the_device_too():
    """The audit of padding rows: positions and ids of the padding are the poison's when the graph runs, and no real row shows them."""
    from cubic_serve_b200.executor.gpu_executor import Segment
    outs = []
    for poison in (False, True):
        ex = _laid_out()
        ex.capture_decode_graphs([4, 8])
        segs = lambda start, n: [Segment(i, [3 + i] * n, start, [2 * i + 1, 2 * i + 2], True, uid=i) for i in range(5)]        # noqa: E731
        ex.execute(segs(0, 20))
        ex.audit_poison_padding = poison
        outs.append((ex.execute(segs(20, 1)).tolist(), ex.logits[:5].clone()))
        torch.cuda.synchronize()
        positions, host = ex.stage.d["positions"][:8].tolist(), ex.stage.h["positions"][5:8].tolist()
        assert positions[:5] == [20] * 5 and ex.stage.d["slots"][5:8].tolist() == [-1] * 3 and ex.stage.d["rb_qcount"][5:8].tolist() == [0] * 3
        if poison:
            assert positions[5:] == host and any(positions[5:]), "the poison reached the device"
        else:
            assert positions[5:] == [0] * 3
    assert outs[0][0] == outs[1][0] and torch.equal(outs[0][1], outs[1][1])


def test_the_graph_audit_of_an_executor_with_layout_on_the_device():
    from cubic_serve_b200.guardrail.graph_audit import audit_decode_graphs
    r = np.random.default_rng(0)
    rep = audit_decode_graphs(_laid_out, [r.integers(0, 1000, 12 + 3 * i).tolist() for i in range(3)], (4, 8))
    assert rep.poisoned_padding_bit_identical and rep.poisoned_padding_finite and rep.permutation_bit_identical


def test_prompts_of_many_rows_are_computed_with_their_adapters(tmp_path):
    """Steps of 700 and 1000 tokens, several adapters and none among them: every prompt's logits are those of a step of its own, within the rounding of
    bf16 activations (three layers, some ten roundings of 2^-8 in a row), which the adapters move by much more."""
    from cubic_serve_b200.executor.gpu_executor import GpuExecutor, Segment
    from cubic_serve_b200.models.decoder import DecoderRunner, random_decoder_weights
    from test_gpu_step_serving import CFG, _adapter
    ranks = (4, 16, 40, 64)
    for i, rank in enumerate(ranks):
        _adapter(tmp_path / f"a{i}", 30 + i, rank=rank, modules=("q_proj", "v_proj", "o_proj", "gate_proj", "down_proj") if i % 2 else ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"))
    runner = DecoderRunner(CFG, random_decoder_weights(CFG, torch.device(DEV), seed=3, std=0.05), num_pages=160, max_tokens=1024, max_requests=8, low_rank=(4, 64))
    ex = GpuExecutor(runner, max_rows=8, max_prefill_tokens=1024, max_model_len=512, use_graphs=False)
    for i in range(4):
        ex.load_adapter(f"a{i}", tmp_path / f"a{i}")
    r = np.random.default_rng(4)
    for lengths, slots in (((150, 90, 201, 160, 99), (0, -1, 3, 1, 2)), ((331, 13, 400, 257), (1, 2, 2, -1))):
        prompts = [r.integers(0, CFG.vocab_size, n).tolist() for n in lengths]
        segs = [Segment(i, p, 0, list(range(1 + 32 * i, 33 + 32 * i)), logit_offsets=[len(p) - 1], adapter=s) for i, (p, s) in enumerate(zip(prompts, slots))]

        def logits(some):
            ex.invalidate_page_rows(range(8))
            return torch.from_numpy(np.concatenate(ex.execute_logits(some)))

        together, alone = logits(segs), torch.cat([logits([s]) for s in segs])
        for s in segs:
            s.adapter = -1
        without = logits(segs)
        off, moved = (together - alone).norm(dim=1) / alone.norm(dim=1), (without - alone).norm(dim=1) / alone.norm(dim=1)
        named = torch.tensor(slots) >= 0
        assert bool((off < 0.1).all()) and bool((moved[named] > 0.3).all()) and bool((moved[~named] < 0.1).all()), (off, moved)


def test_buffers_of_the_layout_are_there_before_the_first_step():
    """Made in the constructor, which waits for the caller's stream: a step's stream writes no memory that the caller's still uses."""
    ex = _laid_out(graphs=False)
    assert ex.builder.given.is_cuda and ex.builder.given.numel() == ex.builder.given_host.numel() >= 8 * (256 // 16 + 1)


@pytest.mark.parametrize("model", ["layered-tiny", "layered-seq-tiny", "layered-streams-tiny", "layered-gated-tiny"])
def test_layered_decoders_are_laid_out_on_the_device_as_on_the_host(model):
    """Layered decoders through the server's engine: prompts in portions, decode, draws from the whole vocabulary."""
    from cubic_serve_b200.cli import build_parser, parse_speculative_config
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    from cubic_serve_b200.runtime.serving import build_backend
    outs = []
    for flags in ((), ("--device-layout",)):
        args = build_parser().parse_args(["serve", f"random:{model}", "--max-running-requests", "6", "--gpu-memory-gib", "8", "--gpu-reserve-gib", "0.5", "--token-budget", "64",
                                          "--prefill-chunk-tokens", "48", "--max-model-len", "256", *flags])
        backend, _ = build_backend(args, [0], 1, parse_speculative_config(None), 8, 8)
        backend.close()
        eng = backend.engine
        assert (eng.executor.layout is not None) == bool(flags)
        r = np.random.default_rng(3)
        ids = [eng.add_request(r.integers(0, 200, int(r.integers(3, 90))).tolist(), SamplingParams(max_tokens=9 + i, ignore_eos=True, seed=i, temperature=0.9 * (i % 2), whole_vocabulary=i % 4 == 1, min_p=0.02 if i % 4 == 3 else 0.0))
               for i in range(9)]
        reqs = [eng.requests[i] for i in ids]
        while eng.has_unfinished:
            eng.step()
        outs.append([list(q.output) for q in reqs])
        assert all(len(q.output) == 9 + i for i, q in enumerate(reqs))
    assert outs[0] == outs[1]


@pytest.mark.parametrize("kind", ["experts", "hybrid"])
def test_decoders_with_experts_and_recurrent_mixers_are_laid_out_on_the_device_as_on_the_host(kind):
    """Prompts in portions, decode and preemption, with draws from the whole vocabulary."""
    from dataclasses import replace

    from test_gpu_step_serving import CFG, _engine, _executor, _prompts, _run, _sampling
    cfg = replace(CFG, family="gqa_moe", num_experts=8, experts_per_token=2, moe_intermediate_size=256, intermediate_size=0) if kind == "experts" else \
        replace(CFG, family="qwen3_5", num_layers=4, gdn_interval=4, gdn_k_heads=2, gdn_v_heads=4, attn_output_gate=True, rotary_dim=64)
    outs = []
    for layout in (False, True):
        eng = _engine(_executor(cfg, device_layout=layout), pages=48, prefill_chunk_tokens=64, enable_prefix_cache=False)
        outs.append(_run(eng, [(p, _sampling(max_tokens=10 + i, seed=i, temperature=0.8 * (i % 2), whole_vocabulary=True)) for i, p in enumerate(_prompts(12, 4, 5, 90))]))
    assert outs[0] == outs[1]


@pytest.mark.parametrize("graphs", [True, False])
def test_steps_laid_out_by_the_host_and_on_the_device_in_turn(graphs):
    """What happens when requests with media come and go: the block table of either side is whole after steps of the other."""
    from test_gpu_step_serving import _engine, _executor, _prompts, _run, _sampling
    requests = [(p, _sampling(max_tokens=14 + i)) for i, p in enumerate(_prompts(12, 14, 5, 90))]
    outs = []
    for mixed in (False, True):
        ex = _executor(graphs=graphs, device_layout=mixed)
        eng = _engine(ex, pages=44, prefill_chunk_tokens=64)
        if mixed:
            launch, layout, turn = ex.launch, ex.layout, np.random.default_rng(2)

            def either(segs, feedback_rows=0):
                ex.layout = layout if turn.random() < 0.6 else None
                return launch(segs, feedback_rows)

            ex.launch = either
        outs.append(_run(eng, requests))
    assert outs[0] == outs[1]
