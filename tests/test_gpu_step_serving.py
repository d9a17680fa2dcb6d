"""Layout on the device, low-rank adapters and whole-vocabulary draws in a served decoder, alone and together."""
import json

import numpy as np
import pytest
import torch

from cubic_serve_b200.models.config import ModelConfig, QuantSpec

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = ModelConfig(name="step-serving", num_layers=3, hidden_size=256, num_q_heads=4, num_kv_heads=2, head_dim=128, intermediate_size=512, vocab_size=1000,
                  rope_theta=1e4, quant=QuantSpec("none"))


def _executor(cfg=CFG, low_rank=None, graphs=True, weights=None, think=None, **kw):
    from cubic_serve_b200.executor.gpu_executor import GpuExecutor
    from cubic_serve_b200.models.decoder import DecoderRunner, random_decoder_weights
    runner = DecoderRunner(cfg, weights or random_decoder_weights(cfg, torch.device(DEV), seed=3, std=0.05), num_pages=96, max_tokens=256, max_requests=8, low_rank=low_rank)
    if think:
        runner.enable_reasoning_budget(*think)
    ex = GpuExecutor(runner, max_rows=8, max_prefill_tokens=256, max_model_len=256, use_graphs=graphs, **kw)
    return ex


def _engine(ex, adapters=(), capture=True, pages=96, **kw):
    from cubic_serve_b200.runtime.engine import LLMEngine
    from cubic_serve_b200.runtime.scheduler import SchedulerConfig
    eng = LLMEngine(ex, num_pages=pages, scheduler_config=SchedulerConfig(max_running_requests=8, max_model_len=256, max_batched_tokens=256, **kw))
    for name, path in adapters:
        eng.load_adapter(name, path)
    if capture and ex.use_graphs:
        ex.capture_decode_graphs([1, 2, 4, 8])
    return eng


def _prompts(n, seed=0, lo=5, hi=70):
    r = np.random.default_rng(seed)
    return [r.integers(0, CFG.vocab_size, int(r.integers(lo, hi))).tolist() for _ in range(n)]


def _run(eng, requests):
    """Tokens of every (prompt, sampling), all admitted at once."""
    ids = [eng.add_request(p, s) for p, s in requests]
    reqs = [eng.requests[i] for i in ids]
    while eng.has_unfinished:
        eng.step()
    return [list(r.output) for r in reqs]


def _sampling(**kw):
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    return SamplingParams(**{"max_tokens": 12, "ignore_eos": True, **kw})


# ------------------------------------------------------------------------------------------------- draws
@pytest.mark.parametrize("graphs", [True, False])
def test_whole_vocabulary_draws_in_the_engine(graphs):
    eng = _engine(_executor(graphs=graphs))
    p = _prompts(6)
    greedy = _run(eng, [(q, _sampling()) for q in p])
    narrow = [_sampling(temperature=0.9, whole_vocabulary=True, top_k=1, seed=5), _sampling(temperature=1.3, min_p=1.0, seed=5), _sampling(),
              _sampling(temperature=0.7, whole_vocabulary=True, top_p=1e-6, seed=9), _sampling(temperature=0.0, whole_vocabulary=True, top_k=500), _sampling()]
    assert _run(eng, list(zip(p, narrow))) == greedy, "prefixes of one token are the largest value"
    wide = [_sampling(temperature=1.5, whole_vocabulary=True, seed=11 + i) for i in range(6)]
    a = _run(eng, list(zip(p, wide)))
    assert a == _run(eng, list(zip(p, wide))) and len({t for o in a for t in o}) > 40, "the same seeds draw the same, from more than a few tokens"
    top20 = [_sampling(temperature=0.8, top_k=20, top_p=0.9, seed=70 + i) for i in range(6)]
    assert _run(eng, list(zip(p, top20))) == _run(eng, [(q, _sampling(temperature=0.8, top_k=20, top_p=0.9, seed=70 + i, whole_vocabulary=True)) for i, q in enumerate(p)])
    mixed = [wide[0], _sampling(), top20[2], _sampling(), wide[4], top20[5]]
    got = _run(eng, list(zip(p, mixed)))
    assert [got[1], got[3]] == [greedy[1], greedy[3]]


def test_whole_vocabulary_draws_before_thinking_budgets():
    """The budget's forced tokens replace what was drawn, in steps that draw from the whole vocabulary as in others."""
    think = (999, [7, 8, 999])
    eng = _engine(_executor(think=think))
    out = _run(eng, [(q, _sampling(temperature=1.5, whole_vocabulary=True, seed=i, thinking_budget=4)) for i, q in enumerate(_prompts(3))])
    for o in out:
        end = o.index(999) if 999 in o[:4] else None
        assert end is not None or o[4:7] == [7, 8, 999]


def test_draws_that_an_executor_does_not_offer_are_refused():
    from cubic_serve_b200.runtime.scheduler import AdmissionError
    ex = _executor(graphs=False)
    ex.accepts_vocabulary_draws = False
    eng = _engine(ex)
    with pytest.raises(AdmissionError):
        eng.add_request([1, 2], _sampling(temperature=1.0, min_p=0.1))
    with pytest.raises(AdmissionError):
        eng.add_request([1, 2], _sampling(adapter="a"))
    eng.add_request([1, 2], _sampling(temperature=0.0, whole_vocabulary=True))


# ------------------------------------------------------------------------------------------------- adapters
def _adapter(path, seed, rank=8, alpha=16, modules=("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"), layers=range(CFG.num_layers), std=0.06, **cfg):
    from safetensors.torch import save_file
    g = torch.Generator().manual_seed(seed)
    D = CFG.head_dim
    shapes = {"q_proj": (CFG.num_q_heads * D, 256), "k_proj": (CFG.num_kv_heads * D, 256), "v_proj": (CFG.num_kv_heads * D, 256), "o_proj": (256, CFG.num_q_heads * D),
              "gate_proj": (512, 256), "up_proj": (512, 256), "down_proj": (256, 512)}
    t = {}
    for i in layers:
        for m in modules:
            n, k = shapes[m]
            part = "self_attn" if m[0] in "qkvo" else "mlp"
            t[f"base_model.model.model.layers.{i}.{part}.{m}.lora_A.weight"] = torch.randn(rank, k, generator=g) * k ** -0.5
            t[f"base_model.model.model.layers.{i}.{part}.{m}.lora_B.weight"] = torch.randn(n, rank, generator=g) * std
    path.mkdir(exist_ok=True)
    save_file(t, str(path / "adapter_model.safetensors"))
    (path / "adapter_config.json").write_text(json.dumps({"r": rank, "lora_alpha": alpha, "bias": "none", **cfg}))
    return t


def _logits(ex, rows):
    """Logits of the last token of every (tokens, adapter slot), one prefill step."""
    from cubic_serve_b200.executor.gpu_executor import Segment
    segs = [Segment(i, t, 0, list(range(1 + 8 * i, 9 + 8 * i)), logit_offsets=[len(t) - 1], adapter=a) for i, (t, a) in enumerate(rows)]
    ex.invalidate_page_rows(range(8))
    return torch.from_numpy(np.concatenate(ex.execute_logits(segs)))


def _merged(tensors, scale):
    from cubic_serve_b200.models.decoder import random_decoder_weights
    from cubic_serve_b200.ops import wq_pack
    w = random_decoder_weights(CFG, torch.device(DEV), seed=3, std=0.05)
    for i, lw in enumerate(w.layers):
        def delta(m):
            part = "self_attn" if m[0] in "qkvo" else "mlp"
            at = f"base_model.model.model.layers.{i}.{part}.{m}."
            return (tensors[at + "lora_B.weight"] @ tensors[at + "lora_A.weight"] * scale).to(DEV)
        for name, mods in (("qkv", "qkv"), ("o", "o"), ("gate_up", ("gate", "up")), ("down", ("down",))):
            d = torch.cat([delta(m + "_proj") for m in mods])
            setattr(lw, name, wq_pack.pack_bf16(wq_pack.unpack_to_dense(getattr(lw, name)).to(DEV)[:d.shape[0]] + d))
    return w


def test_an_adapter_is_its_merged_weights(tmp_path):
    """Against weights with the adapter added: off by the rounding of bf16 activations and weights (2^-8 a value, some ten of them in a row of three
    layers: under a tenth), where the adapter itself changes the logits by about as much as they are."""
    t = _adapter(tmp_path / "a", 1)
    ex = _executor(low_rank=(3, 16), graphs=False)
    ex.load_adapter("a", tmp_path / "a")
    prompts = _prompts(4, 2)
    base, with_a = _logits(ex, [(p, -1) for p in prompts]), _logits(ex, [(p, 0) for p in prompts])
    want = _logits(_executor(graphs=False, weights=_merged(t, 2.0)), [(p, -1) for p in prompts])
    plain = _logits(_executor(graphs=False), [(p, -1) for p in prompts])
    moved, off = (want - plain).norm(dim=1) / plain.norm(dim=1), (with_a - want).norm(dim=1) / want.norm(dim=1)
    assert bool((moved > 0.3).all()) and bool((off < 0.1).all()), (moved, off)
    assert bool(((base - plain).norm(dim=1) / plain.norm(dim=1) < 0.05).all())


def test_a_request_does_not_see_the_adapters_of_others(tmp_path):
    for i in range(3):
        _adapter(tmp_path / f"a{i}", 10 + i, rank=(4, 16, 9)[i], modules=(("q_proj", "down_proj"), ("v_proj", "o_proj", "gate_proj"), ("up_proj",))[i])
    ex = _executor(low_rank=(4, 16), graphs=False)
    for i in range(3):
        ex.load_adapter(f"a{i}", tmp_path / f"a{i}")
    p = _prompts(6, 3)
    first = _logits(ex, list(zip(p, [0, 1, -1, 2, 0, -1])))
    other = _logits(ex, list(zip(p, [0, 2, -1, 1, 1, 3])))
    same = [0, 2]
    assert torch.equal(first[same], other[same]) and not any(torch.equal(first[i], other[i]) for i in (1, 3, 4))
    assert torch.equal(first[5], other[5]), "an empty slot is no adapter"


def test_adapters_in_the_engine_decode_in_graphs_and_share_no_prefix(tmp_path):
    _adapter(tmp_path / "a", 1)
    _adapter(tmp_path / "b", 2, rank=16, use_rslora=True)
    adapters = [("a", tmp_path / "a"), ("b", tmp_path / "b")]
    prompt = _prompts(1, 9, 60, 64)[0]
    fresh = {}
    for name in (None, "a", "b"):
        eng = _engine(_executor(low_rank=(2, 16)), adapters)
        fresh[name] = _run(eng, [(prompt, _sampling(adapter=name))])[0]
        assert _run(eng, [(prompt, _sampling(adapter=name))])[0] == fresh[name] and eng.prefix.hit_tokens > 0, "its own prefix is shared"
    assert len({tuple(v) for v in fresh.values()}) == 3
    eng = _engine(_executor(low_rank=(2, 16)), adapters)
    for name, again in ((None, False), ("b", False), ("a", False), (None, True), ("b", True)):
        hits = eng.prefix.hit_tokens
        assert _run(eng, [(prompt, _sampling(adapter=name))])[0] == fresh[name]
        assert (eng.prefix.hit_tokens > hits) == again, "a prefix computed with another adapter is not taken"
    assert len(eng.executor.graphs) == 4


def test_adapters_are_loaded_and_unloaded_between_steps(tmp_path):
    from cubic_serve_b200.models.low_rank import AdapterError
    from cubic_serve_b200.runtime.scheduler import AdmissionError
    _adapter(tmp_path / "a", 1)
    _adapter(tmp_path / "big", 2, rank=32)
    _adapter(tmp_path / "far", 3, layers=range(1, 5))
    eng = _engine(_executor(low_rank=(1, 16)))
    p = _prompts(2, 4)
    base = _run(eng, [(q, _sampling()) for q in p])
    for bad in ("big", "far", "missing"):
        with pytest.raises(AdapterError):
            eng.load_adapter(bad, tmp_path / bad)
    assert _run(eng, [(q, _sampling()) for q in p]) == base and eng.adapter_names == ()
    eng.load_adapter("a", tmp_path / "a")
    with pytest.raises(AdapterError):
        eng.load_adapter("b", tmp_path / "a")
    rid = eng.add_request(p[0], _sampling(adapter="a"))
    eng.step()
    with pytest.raises(AdmissionError):
        eng.unload_adapter("a")
    first = eng.requests[rid]
    while eng.has_unfinished:
        eng.step()
    eng.unload_adapter("a")
    with pytest.raises(AdmissionError):
        eng.add_request(p[0], _sampling(adapter="a"))
    assert _run(eng, [(q, _sampling()) for q in p]) == base
    eng.load_adapter("again", tmp_path / "a")
    assert _run(eng, [(p[0], _sampling(adapter="again"))])[0] == first.output


def test_adapters_beside_fp8_and_packed_weights(tmp_path):
    """Projections whose input is quantized by the norm in front of them get their rows unquantized for the adapters."""
    from dataclasses import replace
    _adapter(tmp_path / "a", 1)
    for quant in (QuantSpec("fp8", 8, 0), QuantSpec("cubic", 4, 128)):
        cfg = replace(CFG, quant=quant)
        ex = _executor(cfg, low_rank=(2, 16), graphs=False)
        ex.load_adapter("a", tmp_path / "a")
        p = _prompts(3, 5)
        mixed, none = _logits(ex, list(zip(p, (0, -1, 0)))), _logits(ex, [(q, -1) for q in p])
        plain = _logits(_executor(cfg, graphs=False), [(q, -1) for q in p])
        assert bool(((none - plain).norm(dim=1) / plain.norm(dim=1) < 0.1).all()) and torch.equal(mixed[1], none[1])
        assert bool((((mixed - none).norm(dim=1) / none.norm(dim=1))[[0, 2]] > 0.3).all())


@pytest.mark.parametrize("kind", ["experts", "hybrid"])
def test_adapters_of_attention_layers_beside_experts_and_recurrent_mixers(tmp_path, kind):
    from dataclasses import replace

    from cubic_serve_b200.models.low_rank import AdapterError
    if kind == "experts":
        cfg = replace(CFG, family="gqa_moe", num_experts=8, experts_per_token=2, moe_intermediate_size=256, intermediate_size=0)
    else:
        cfg = replace(CFG, family="qwen3_5", num_layers=4, gdn_interval=4, gdn_k_heads=2, gdn_v_heads=4, attn_output_gate=True, rotary_dim=64)
    full = [i for i in range(cfg.num_layers) if not cfg.layer_is_gdn(i)]
    _adapter(tmp_path / "a", 1, modules=("q_proj", "v_proj", "o_proj"), layers=full)
    _adapter(tmp_path / "no", 1, modules=("gate_proj",) if kind == "experts" else ("q_proj",), layers=range(cfg.num_layers))
    ex = _executor(cfg, low_rank=(2, 8))
    with pytest.raises(AdapterError):
        ex.load_adapter("no", tmp_path / "no")
    eng = _engine(ex, [("a", tmp_path / "a")], enable_prefix_cache=False)
    p = _prompts(4, 7)
    none = _run(eng, [(q, _sampling()) for q in p])
    mixed = _run(eng, [(q, _sampling(adapter="a" if i % 2 else None)) for i, q in enumerate(p)])
    assert [mixed[0], mixed[2]] == [none[0], none[2]] and mixed[1] != none[1] and mixed[3] != none[3]
    if kind == "experts":
        assert none == _run(_engine(_executor(cfg), enable_prefix_cache=False), [(q, _sampling()) for q in p]), "without an adapter the model is what it was"


# ------------------------------------------------------------------------------------------------- layout
def _compare_layout(ex, seen):
    """After every launch what the device made is what the host would have filled in."""
    from cubic_serve_b200.executor.gpu_executor import BatchBuilder
    launch, n = ex.launch, ex.builder
    host = BatchBuilder(n.max_rows, n.max_tokens, 256, 16 // n.qb, n.kv_heads, "cpu")

    def checked(segs, feedback_rows=0):
        handle = launch(segs, feedback_rows)
        torch.cuda.synchronize()
        t = sum(len(s.token_ids) for s in segs)
        cap = ex.graph_rt.dispatch(t) if all(len(s.token_ids) == 1 for s in segs) and ex.use_graphs else None
        host.invalidate_page_rows([s.request_slot for s in segs])
        b, _ = host._fill(segs, pad_rows_to=cap)
        h, d = host.stage.h, ex.stage.d
        for name, k in (("positions", b.num_tokens), ("slots", b.num_tokens), ("rb_req", b.num_row_blocks), ("rb_qstart", b.num_row_blocks), ("rb_qcount", b.num_row_blocks),
                        ("rb_ctx", b.num_row_blocks), ("seg_row0", len(segs)), ("logit_rows", b.num_logit_rows)):
            assert d[name][:k].cpu().numpy().tolist() == h[name][:k].tolist(), name
        for s in segs:
            k = -(-(s.start + len(s.token_ids)) // 16)
            assert d["page_table"][s.request_slot, :k].tolist() == list(s.pages[:k])
        assert ex.layout.totals.tolist()[3] == 0
        seen.append((t, handle["h2d"]))
        return handle

    ex.launch = checked


@pytest.mark.parametrize("graphs", [True, False])
def test_layout_on_the_device_is_the_hosts(graphs):
    """Prefill in portions, decode, shared prefixes, preemption and slots that change hands."""
    r = np.random.default_rng(1)
    shared = r.integers(0, CFG.vocab_size, 48).tolist()
    requests = [(shared + q if i % 2 else q, _sampling(max_tokens=20 + 3 * i)) for i, q in enumerate(_prompts(14, 6, 5, 90))]
    outs, seen = [], []
    for device in (False, True):
        ex = _executor(graphs=graphs, device_layout=device)
        eng = _engine(ex, pages=40, prefill_chunk_tokens=64)
        if device:
            _compare_layout(ex, seen)
        ids = [eng.add_request(q, s) for q, s in requests]
        reqs = [eng.requests[i] for i in ids]
        while eng.has_unfinished:
            eng.step()
        outs.append([r.output for r in reqs])
        assert sum(r.preemptions for r in reqs) > 0 and eng.prefix.hit_tokens > 0
    assert outs[0] == outs[1]
    assert len({t for t, _ in seen}) > 3 and max(b for _, b in seen) < ex.stage.nbytes / 2


def test_everything_around_a_step_together(tmp_path):
    """Layout on the device, adapters, whole-vocabulary draws, a grammar-like mask and greedy rows in the same steps."""
    for i in range(3):
        _adapter(tmp_path / f"a{i}", 20 + i, rank=4 + 4 * i)
    adapters = [(f"a{i}", tmp_path / f"a{i}") for i in range(3)]
    p = _prompts(12, 8)
    kinds = [dict(), dict(adapter="a0"), dict(temperature=1.2, whole_vocabulary=True, seed=1), dict(temperature=0.9, min_p=0.05, adapter="a1", seed=2),
             dict(temperature=0.8, top_k=10, adapter="a2", seed=3), dict(temperature=1.0, whole_vocabulary=True, top_k=300, top_p=0.95, adapter="a0", seed=4)]
    requests = [(q, _sampling(max_tokens=10 + i, **kinds[i % 6])) for i, q in enumerate(p)]
    outs = []
    for device in (False, True):
        ex = _executor(low_rank=(4, 16), device_layout=device)
        outs.append(_run(_engine(ex, adapters, pages=48, prefill_chunk_tokens=64), requests))
        ex.runner.ws.check_status()
    assert outs[0] == outs[1] and all(len(o) == 10 + i for i, o in enumerate(outs[0]))
