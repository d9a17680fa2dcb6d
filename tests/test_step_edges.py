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


# ------------------------------------------------------------------------------------------------- memory of a deployment with adapters
def _planned_pages(monkeypatch, model, free, *flags):
    """KV pages that a server would plan with so many bytes free, and the layers it would serve."""
    from types import SimpleNamespace

    from cubic_serve_b200.cli import build_parser, parse_speculative_config
    from cubic_serve_b200.models import registry
    from cubic_serve_b200.models.config import NAMED_CONFIGS
    from cubic_serve_b200.runtime.serving import build_backend

    cfg = NAMED_CONFIGS[model]()
    layers = [SimpleNamespace(gdn=object() if cfg.layer_is_gdn(i) else None, moe=object() if cfg.is_moe else None) for i in range(cfg.num_layers)]

    class Planned(Exception):
        pass

    def runner(*_, num_pages, **kw):
        raise Planned(num_pages)

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda d: (free, free))
    monkeypatch.setattr(registry, "get", lambda family: SimpleNamespace(random_weights=lambda *a: SimpleNamespace(layers=layers), build_runner=runner))
    args = build_parser().parse_args(["serve", f"random:{model}", "--max-running-requests", "256", "--max-model-len", "32768", "--token-budget", "8192", *flags])
    with pytest.raises(Planned) as got:
        build_backend(args, [0], 1, parse_speculative_config(None), 8, 8)
    return got.value.args[0], cfg, layers


@pytest.mark.parametrize("model,slots,rank", [("dense-8b", 16, 64), ("dense-8b", 64, 64), ("moe-30b-a3b", 5, 20), ("hybrid-8b", 3, 128)])
def test_the_kv_cache_leaves_room_for_the_adapters(monkeypatch, model, slots, rank):
    from cubic_serve_b200.contracts.model import CacheSpec
    flags = ("--low-rank-slots", str(slots), "--low-rank-max-rank", str(rank))
    without, cfg, layers = _planned_pages(monkeypatch, model, 60 << 30)
    with_them, _, _ = _planned_pages(monkeypatch, model, 60 << 30, *flags)
    # every slot has A and B of each projection, ranks stored as 16, 32, 64 or 128; h of a step's rows
    stored, D = next(r for r in (16, 32, 64, 128) if r >= rank), cfg.head_dim
    q, kv, h, i = cfg.num_q_heads * D, cfg.num_kv_heads * D, cfg.hidden_size, cfg.intermediate_size
    need = 0
    for lw in layers:
        if lw.gdn is None:
            need += (3 * h + q + 2 * kv) + (q + h)
        if lw.moe is None:
            need += (2 * h + 2 * i) + (i + h)
    need = need * slots * stored * 2 + 2 * 2 * 8192 * 3 * stored
    page = CacheSpec(sum(lw.gdn is None for lw in layers), cfg.num_kv_heads, D, 8, 8).page_bytes
    assert need / page <= without - with_them <= need / page * 1.02 + 2, "pages given up are the adapters' bytes, and their rows' lists"


def test_adapters_that_leave_no_room_are_refused(monkeypatch):
    with pytest.raises(SystemExit, match="GiB"):
        _planned_pages(monkeypatch, "dense-8b", 20 << 30, "--low-rank-slots", "64")


def test_empty_banks_take_their_own_memory_and_no_more():
    """The sum that a server plans with is what the banks hold."""
    from types import SimpleNamespace

    from cubic_serve_b200.models.config import ModelConfig, QuantSpec
    from cubic_serve_b200.models.low_rank import LowRankAdapters
    cfg = ModelConfig(name="t", num_layers=2, hidden_size=72, num_q_heads=2, num_kv_heads=1, head_dim=32, intermediate_size=96, vocab_size=128, quant=QuantSpec("none"))
    layers = [SimpleNamespace(gdn=None, moe=None), SimpleNamespace(gdn=None, moe=object())]
    real, planned = LowRankAdapters(cfg, layers, 3, 20, 50, "cpu"), LowRankAdapters(cfg, layers, 3, 20, 50, "meta")
    held = [t for banks in real.banks for b in banks.values() for t in vars(b).values() if isinstance(t, torch.Tensor)] + [t for t in vars(real.rows).values() if isinstance(t, torch.Tensor)]
    assert planned.nbytes == real.nbytes == sum(t.untyped_storage().nbytes() for t in held)
    assert not any(t.any() for t in held)


def test_adapters_of_a_family_without_a_native_runner_are_refused(monkeypatch):
    """Not left out in silence: a request that names one would be told that there is no such model."""
    from cubic_serve_b200.cli import build_parser, parse_speculative_config
    from cubic_serve_b200.runtime.serving import build_backend
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    args = build_parser().parse_args(["serve", "random:qwen4-exp-tiny", "--low-rank-slots", "2", "--execution-mode", "cuda"])
    with pytest.raises(SystemExit, match="low-rank adapters"):
        build_backend(args, [0], 1, parse_speculative_config(None), 8, 8)


# ------------------------------------------------------------------------------------------------- steps laid out on the device
def test_a_step_that_lacks_pages_is_not_staged_for_the_device():
    """As the host's layout: an error before anything is launched, and what the device's rows hold is still known."""
    from cubic_serve_b200.executor.gpu_executor import BatchBuilder, Segment
    b = BatchBuilder(4, 128, 96, 4, 2, "cpu")                         # six pages a row
    good = Segment(0, [1] * 20, 0, [7, 8], True, uid=5)

    def stage(*segs):
        b._fill(list(segs), lengths=True)
        n = b.stage_layout(list(segs))
        return b.given_host[:len(segs) + n].tolist()

    assert stage(good) == [0, 7, 8]
    for bad in (Segment(1, [1], 16, [3], True, uid=6), Segment(1, [1] * 40, 0, [3, 4], True, uid=6), Segment(1, [1] * 3, 30, [], True, uid=6),
                Segment(1, [1], 96, list(range(20, 27)), True, uid=6), Segment(1, [1] * 60, 50, list(range(20, 27)), True, uid=6)):
        for order in ((bad, good), (good, bad)):
            with pytest.raises(IndexError, match="pages"):
                stage(*order)
    assert stage(Segment(0, [1], 20, [7, 8], True, uid=5)) == [2] and stage(Segment(0, [1] * 13, 21, [7, 8, 9], True, uid=5)) == [2, 9]
    assert stage(Segment(1, [1], 95, list(range(20, 26)), True, uid=6), Segment(0, [1], 34, [7, 8, 9], True, uid=5)) == [0, 3, *range(20, 26)]


# ------------------------------------------------------------------------------------------------- requests
def test_whole_vocabulary_requests_are_not_cut_to_the_checkpoints_top_k():
    """A checkpoint's recommended ``top_k`` (kept as 20 at most, for the sampler of 20) is the default of requests to that sampler alone."""
    from cubic_serve_b200.inputs.normalize import normalize_openai_chat_completions as n
    body, defaults = {"model": "m", "messages": [{"role": "user", "content": "x"}]}, {"temperature": 0.6, "top_p": 0.95, "top_k": 20}
    top_k = lambda **kw: n({**body, **kw}, "m", defaults).sampling.top_k        # noqa: E731
    assert top_k() == 20 and top_k(min_p=0.0) == 20 and top_k(whole_vocabulary=False) == 20 and top_k(min_p=None) == 20
    assert top_k(whole_vocabulary=True) == 0 and top_k(min_p=0.05) == 0 and top_k(whole_vocabulary=True, top_k=None) == 0
    assert top_k(whole_vocabulary=True, top_k=300) == 300 and top_k(min_p=0.05, top_k=7) == 7 and top_k(whole_vocabulary=True, top_k=0) == 0
    s = n({**body, "whole_vocabulary": True}, "m", defaults).sampling
    assert (s.temperature, s.top_p) == (0.6, 0.95), "what else the checkpoint recommends holds"
