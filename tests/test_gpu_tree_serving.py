"""Penalties, biases and drafts in trees through the engine."""
import numpy as np
import pytest
import torch

from cubic_serve_b200.models.config import ModelConfig, QuantSpec

pytestmark = pytest.mark.gpu
VOCAB = 2048


def _engine(kind="plain", graphs=True, max_rows=8, seed=0, kb=8, vb=8, rotation=False, reasoning=None, **kw):
    from cubic_serve_b200.executor.gpu_executor import GpuExecutor
    from cubic_serve_b200.executor.spec_executor import NgramSpeculativeGpuExecutor, NgramTreeSpeculativeGpuExecutor
    from cubic_serve_b200.models.decoder import DecoderRunner, random_decoder_weights
    from cubic_serve_b200.runtime.engine import LLMEngine
    from cubic_serve_b200.runtime.scheduler import SchedulerConfig
    dev = torch.device("cuda")
    cfg = ModelConfig(name="tree", num_layers=2, hidden_size=512, num_q_heads=8, num_kv_heads=2, head_dim=128, intermediate_size=1024, vocab_size=VOCAB, rope_theta=1e6,
                      qk_norm=True, quant=QuantSpec("cubic", 4, 128))
    runner = DecoderRunner(cfg, random_decoder_weights(cfg, dev, seed=seed, std=0.05), num_pages=256, max_tokens=512, k_bits=kb, v_bits=vb, kv_rotation=rotation)
    if reasoning:
        runner.enable_reasoning_budget(*reasoning)
    make = {"plain": lambda **k: GpuExecutor(runner, use_graphs=graphs, **k), "chain": lambda **k: NgramSpeculativeGpuExecutor(runner, 3, **k),
            "tree": lambda **k: NgramTreeSpeculativeGpuExecutor(runner, 3, 4, **k)}[kind]
    ex = make(max_rows=max_rows, max_prefill_tokens=512, max_model_len=256)
    if graphs:
        ex.capture_decode_graphs([4, 8])
    return LLMEngine(ex, 256, SchedulerConfig(max_running_requests=max_rows, max_model_len=256, max_batched_tokens=512, enable_prefix_cache=kw.get("prefix", False))), ex, runner


def _sampling(**kw):
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    return SamplingParams(**{"max_tokens": 20, "ignore_eos": True, **kw})


def _run(eng, requests):
    ids = [eng.add_request(p, s) for p, s in requests]
    reqs = [eng.requests[i] for i in ids]
    while eng.has_unfinished:
        eng.step()
    return [r.output for r in reqs]


def _prompts(n, seed=3, times=4):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, VOCAB, int(rng.integers(5, 14))).tolist() * times for _ in range(n)]


def _adjusted(logits, tokens, prompt, s):
    x = logits.astype(np.float64).copy()
    for t in set(tokens):
        x[t] = x[t] / s.repetition_penalty if x[t] > 0 else x[t] * s.repetition_penalty
    for t in set(tokens[prompt:]):
        x[t] -= tokens[prompt:].count(t) * s.frequency_penalty + s.presence_penalty
    for t, v in s.logit_bias:
        x[t] += v
    return x


@pytest.mark.parametrize("kind,graphs", [("plain", False), ("plain", True), ("tree", True)])
def test_greedy_tokens_are_the_best_of_the_adjusted_logits(kind, graphs):
    """Every token against logits read anew for its context: the largest after adjustment, to two bf16 steps of the logits' size (another route and batch
    computes them)."""
    from cubic_serve_b200.executor.gpu_executor import Segment
    eng, ex, runner = _engine(kind, graphs)
    wishes = [_sampling(repetition_penalty=1.3), _sampling(frequency_penalty=0.7, presence_penalty=0.5), _sampling(), _sampling(logit_bias=((7, 3.0), (11, -100.0), (1500, 2.5))),
              _sampling(repetition_penalty=0.8, presence_penalty=1.0, logit_bias=((3, 1.0),))]
    prompts = _prompts(5)
    out = _run(eng, list(zip(prompts, wishes)))
    runner.ws.check_status()
    plain, pex, _ = _engine("plain", False)
    for p, s, o in zip(prompts, wishes, out):
        assert len(o) == 20
        seq = p + o
        pages = list(range(-(-len(seq) // 16)))
        offs = list(range(len(p) - 1, len(seq) - 1))
        logits = pex.execute_logits([Segment(0, seq, 0, pages, True, uid=-1, logit_offsets=offs)])[0]
        for k, t in enumerate(o):
            x = _adjusted(logits[k], seq[:len(p) + k], len(p), s)
            assert x[t] >= x.max() - 2 * 2.0 ** -7 * np.abs(logits[k]).max() * max(s.repetition_penalty, 1 / s.repetition_penalty), (k, t, int(x.argmax()))


@pytest.mark.parametrize("kind", ["plain", "tree"])
def test_biases_force_and_forbid(kind):
    eng, ex, runner = _engine(kind)
    p = _prompts(3)
    base = _run(eng, [(q, _sampling()) for q in p])
    forced = _run(eng, [(q, _sampling(logit_bias=((42, 100.0),))) for q in p])
    assert all(set(o) == {42} for o in forced)
    banned = sorted({t for o in base for t in o})
    out = _run(eng, [(q, _sampling(logit_bias=tuple((t, -100.0) for t in banned))) for q in p])
    assert not {t for o in out for t in o} & set(banned)
    assert _run(eng, [(q, _sampling()) for q in p]) == base                                   # nothing stays behind
    once = _run(eng, [(q, _sampling(presence_penalty=2.0, frequency_penalty=2.0, logit_bias=((42, 9.0),))) for q in p])
    assert all(o.count(42) >= 1 for o in once) and all(o.count(42) < 20 for o in once)
    runner.ws.check_status()


def test_graphs_captured_behind_an_adjusted_step_hold_none_of_it():
    eng, ex, runner = _engine()
    p = _prompts(3)
    base = _run(eng, [(q, _sampling()) for q in p])
    assert all(set(o) == {42} for o in _run(eng, [(q, _sampling(logit_bias=((42, 100.0),))) for q in p]))
    ex.capture_decode_graphs([4, 8])
    assert _run(eng, [(q, _sampling()) for q in p]) == base
    assert all(set(o) == {42} for o in _run(eng, [(q, _sampling(logit_bias=((42, 100.0),))) for q in p]))
    runner.ws.check_status()


@pytest.mark.parametrize("kb,vb,rotation", [(8, 8, False), (4, 8, True), (6, 6, False)])
def test_tree_rounds_match_plain_greedy_and_accept_repetitions(kb, vb, rotation):
    eng, _, r0 = _engine("plain", kb=kb, vb=vb, rotation=rotation)
    eng2, ex, runner = _engine("tree", kb=kb, vb=vb, rotation=rotation)
    prompts = _prompts(5)
    plain, spec = (_run(e, [(p, _sampling(max_tokens=40)) for p in prompts]) for e in (eng, eng2))
    runner.ws.check_status()
    assert all(len(o) == 40 for o in spec)
    # Keys and values that another batch computed may be rounded to the neighbouring code, a step of 1 / (2^(bits - 1) - 1) of their group's largest: where two outputs
    # part, the logits of the two tokens are no further apart than that part of the logits' size
    from cubic_serve_b200.executor.gpu_executor import Segment
    _, pex, _ = _engine("plain", False, kb=kb, vb=vb, rotation=rotation)
    for p, x, y in zip(prompts, plain, spec):
        at = next((i for i, (u, v) in enumerate(zip(x, y)) if u != v), None)
        if at is not None:
            seq = p + x[:at]
            logits = pex.execute_logits([Segment(0, seq, 0, list(range(-(-len(seq) // 16))), True, uid=-1, logit_offsets=[len(seq) - 1])])[0][0]
            assert abs(logits[x[at]] - logits[y[at]]) <= np.abs(logits).max() / (2 ** (min(kb, vb) - 1) - 1), (at, logits[x[at]], logits[y[at]])
    s = ex.stats
    assert s["rounds"] > 0 and 0 < s["accepted"] <= s["proposed"]
    assert eng2.pool.num_used == 0


def test_tree_rounds_accept_what_their_drafts_say():
    """A model that is made to say one token over and over is drafted and accepted to the full depth, and its cache stays right: freed of the bias it goes on as
    a plain engine does."""
    eng, ex, runner = _engine("tree")
    p = _prompts(2)
    out = _run(eng, [(q, _sampling(max_tokens=33, logit_bias=((42, 100.0),))) for q in p])
    assert all(o == [42] * 33 for o in out)
    assert ex.stats["accepted"] >= 2 * 3 * 5 and eng.steps < 30


def test_a_tree_executor_takes_sampling_and_constrained_requests_in_plain_steps():
    eng, ex, runner = _engine("tree")
    p = _prompts(3)
    out = _run(eng, [(p[0], _sampling(temperature=0.8, seed=4, repetition_penalty=1.2)), (p[1], _sampling()), (p[2], _sampling(temperature=1.0, seed=5))])
    assert all(len(o) == 20 for o in out)
    other, _, _ = _engine("plain")
    want = _run(other, [(p[0], _sampling(temperature=0.8, seed=4, repetition_penalty=1.2)), (p[1], _sampling()), (p[2], _sampling(temperature=1.0, seed=5))])
    assert np.mean([a == b for x, y in zip(out, want) for a, b in zip(x, y)]) >= 0.9


def test_penalties_before_thinking_budgets():
    """Forced tokens come out as they are, whatever the penalties say of them."""
    eng, ex, runner = _engine("plain", reasoning=(5, [6, 5]))
    out = _run(eng, [(p, _sampling(thinking_budget=4, repetition_penalty=1.5, logit_bias=((6, -100.0), (5, -100.0)))) for p in _prompts(2)])
    assert all(o[4:6] == [6, 5] for o in out)


def test_executors_without_adjustments_refuse():
    from cubic_serve_b200.runtime.scheduler import AdmissionError
    eng, _, _ = _engine("chain")
    for kw in (dict(repetition_penalty=1.1), dict(logit_bias=((1, 1.0),)), dict(presence_penalty=0.1), dict(frequency_penalty=-0.1)):
        with pytest.raises(AdmissionError):
            eng.add_request([1, 2, 3], _sampling(**kw))
    eng, _, _ = _engine("plain")
    with pytest.raises(AdmissionError):
        eng.add_request([1, 2, 3], _sampling(logit_bias=((VOCAB, 1.0),)))


def test_drafts_near_the_end_of_the_model_length_and_of_requests():
    eng, ex, runner = _engine("tree")
    rng = np.random.default_rng(1)
    base = rng.integers(0, VOCAB, 12).tolist()
    p = (base * 21)[:248]
    out = _run(eng, [(p, _sampling(max_tokens=50)), (p[:17], _sampling(max_tokens=1)), (p[:40], _sampling(max_tokens=2))])
    assert [len(o) for o in out] == [8, 1, 2]
    runner.ws.check_status()
    assert eng.pool.num_used == 0


@pytest.mark.parametrize("kind", ["plain", "tree"])
@pytest.mark.parametrize("length,accepts", [((1 << 20) - 300, True), (1 << 20, False)])
def test_engines_of_longer_texts_than_penalties_look_at_refuse_them_at_once(kind, length, accepts):
    from cubic_serve_b200.executor.gpu_executor import GpuExecutor
    from cubic_serve_b200.executor.spec_executor import NgramTreeSpeculativeGpuExecutor
    from cubic_serve_b200.runtime.engine import LLMEngine
    from cubic_serve_b200.runtime.scheduler import AdmissionError, SchedulerConfig
    _, _, runner = _engine("plain", False)
    kw = dict(max_rows=2, max_prefill_tokens=64, max_model_len=length)
    ex = GpuExecutor(runner, use_graphs=False, **kw) if kind == "plain" else NgramTreeSpeculativeGpuExecutor(runner, 3, 4, use_graphs=False, **kw)
    eng = LLMEngine(ex, 256, SchedulerConfig(max_running_requests=2, max_model_len=length, max_batched_tokens=64, enable_prefix_cache=False))
    assert ex.accepts_adjustments == accepts
    wish = _sampling(max_tokens=3, logit_bias=((42, 100.0),))
    if accepts:
        assert _run(eng, [([1, 2, 3], wish)]) == [[42] * 3]
    else:
        with pytest.raises(AdmissionError):
            eng.add_request([1, 2, 3], wish)
    assert len(_run(eng, [([1, 2, 3], _sampling(max_tokens=3))])[0]) == 3
    runner.ws.check_status()


def test_plain_steps_of_a_tree_executor_upload_no_more_than_others():
    """The staging of 4 x 4 drafts a request: its plain steps upload a row of pages a request, and masks have a row a request."""
    from cubic_serve_b200.executor.gpu_executor import GpuExecutor
    from cubic_serve_b200.executor.spec_executor import NgramTreeSpeculativeGpuExecutor
    _, _, runner = _engine("plain", False)
    kw = dict(max_rows=64, max_prefill_tokens=512, max_model_len=4096)
    plain, tree = GpuExecutor(runner, **kw), NgramTreeSpeculativeGpuExecutor(runner, 4, 4, **kw)
    tree.capture_decode_graphs([4])
    assert tree._mask_dev.shape[0] == 64
    # two more pages a row for the drafts, and a row more; the arrays of sampled rows and of row blocks have 512 and 640 entries, of 68 and 16 bytes
    assert tree.stage.nbytes <= plain.stage.nbytes + 4 * (65 * 258 - 64 * 256) + 96 * 512


def test_rounds_take_no_memory_of_their_own_for_their_logits():
    eng, ex, runner = _engine("tree")
    at = ex._rl.data_ptr()
    assert ex._rl.shape == (8 * 13, VOCAB)
    _run(eng, [(q, _sampling(max_tokens=33, logit_bias=((42, 100.0),))) for q in _prompts(8)])
    assert ex.stats["rounds"] > 0 and ex._rl.data_ptr() == at and ex._rl.shape == (8 * 13, VOCAB)


@pytest.mark.parametrize("kb,vb,rotation", [(8, 8, False), (4, 8, True)])
def test_what_rounds_leave_in_the_cache_is_read_on(kb, vb, rotation):
    """Rounds of a biased token, whose drafts branch: most are wrong, some right ones lie behind wrong ones and move up, pages are lent and change hands.  Requests that
    then go on from the cached texts without the bias say what logits of a plain pass over the whole text say, to the rounding of codes and logits."""
    from cubic_serve_b200.executor.gpu_executor import Segment
    eng, ex, runner = _engine("tree", kb=kb, vb=vb, rotation=rotation, prefix=True)
    rng, prompts = np.random.default_rng(8), []
    for i in range(6):
        x = rng.integers(50, VOCAB, 40).tolist()
        prompts.append([42] * 5 + x[:9] + [42, 42] + x[9:20] + [42] * 3 + x[20:20 + 3 * i] + [42, 42])
    moved, keep = [], ex.execute_speculative

    def recorded(segs, **kw):
        out = keep(segs, **kw)
        if ex.last_round["depth"]:
            moved.extend(int(p[k]) != k for p, a in zip(ex._path.cpu().numpy(), ex.last_round["accepted"]) for k in range(1, a + 1))
        return out
    ex.execute_speculative = recorded
    out = _run(eng, [(p, _sampling(max_tokens=30, logit_bias=((42, 100.0),))) for p in prompts])
    assert all(o == [42] * 30 for o in out) and sum(moved) >= len(prompts) and ex.stats["accepted"] < ex.stats["proposed"]
    texts = [p + o[:29] for p, o in zip(prompts, out)]
    ids = [eng.add_request(t, _sampling(max_tokens=12)) for t in texts]
    reqs = [eng.requests[i] for i in ids]
    while eng.has_unfinished:
        eng.step()
    runner.ws.check_status()
    _, pex, _ = _engine("plain", False, kb=kb, vb=vb, rotation=rotation)
    for text, prompt, r in zip(texts, prompts, reqs):
        assert r.num_cached_prefix == (len(text) - 1) // 16 * 16 > len(prompt) + 8             # lines that rounds wrote and moved
        seq = text + r.output
        offs = list(range(len(text) - 1, len(seq) - 1))
        logits = pex.execute_logits([Segment(0, seq, 0, list(range(-(-len(seq) // 16))), True, uid=-1, logit_offsets=offs)])[0]
        for x, t in zip(logits, r.output):
            assert x[t] >= x.max() - np.abs(x).max() / (2 ** (min(kb, vb) - 1) - 1)


@pytest.mark.parametrize("graphs", [True, False])
def test_steps_with_penalties_and_thinking_budgets_replay_their_graphs(graphs):
    """A budget counts what is drawn from the adjusted logits, once: tokens that a bias forces, an end that it brings, and neighbours that want nothing."""
    eng, ex, runner = _engine("plain", graphs, reasoning=(5, [6, 5]))
    p = _prompts(5)
    out = _run(eng, [(p[0], _sampling(thinking_budget=7, logit_bias=((42, 100.0),))), (p[1], _sampling(thinking_budget=3)), (p[2], _sampling(thinking_budget=9, logit_bias=((5, 100.0),))),
                     (p[3], _sampling(thinking_budget=0, logit_bias=((42, 100.0),))), (p[4], _sampling(logit_bias=((43, 100.0),)))])
    assert out[0] == [42] * 7 + [6, 5] + [42] * 11 and out[1][3:5] == [6, 5]
    assert out[2] == [5] * 20 and out[3] == [6, 5] + [42] * 18 and out[4] == [43] * 20
    if graphs:
        assert sum(s["replays"] for s in ex.graph_rt.stats()["slots"].values()) == 19                 # all but the prompts' step
    runner.ws.check_status()


def test_more_requests_than_a_round_takes_run_plainly(monkeypatch):
    from cubic_serve_b200.ops import kernels as K
    monkeypatch.setattr(K, "TREE_MAX_REQUESTS", 4)
    eng, ex, runner = _engine("tree")
    p = _prompts(6)
    wish = [_sampling(max_tokens=n, logit_bias=((42, 100.0),)) for n in (12, 12, 12, 12, 30, 30)]
    assert _run(eng, list(zip(p, wish))) == [[42] * s.max_tokens for s in wish]
    assert ex.stats["rounds"] > 0 and eng.steps >= 12 + 2
    runner.ws.check_status()


def test_rounds_wait_for_constrained_and_sampling_requests():
    """Beside a greedy request that repeats itself: as long as one with a grammar, or one that samples, runs, steps are plain ones, and the grammar holds."""
    from cubic_serve_b200.generation.constraints import ChoiceMatcher

    class Tok:
        def encode(self, text, add_special_tokens=False):
            return [100 + ord(c) for c in text]

    for other in ("grammar", "sampling"):
        eng, ex, runner = _engine("tree")
        p, eos = _prompts(2), 3
        options = ["alpha beta gamma", "alphabet soup, hot"]
        sampling = _sampling(max_tokens=30, ignore_eos=False, stop_token_ids=(eos,), matcher=ChoiceMatcher(options, Tok(), eos), presence_penalty=0.5) if other == "grammar" \
            else _sampling(max_tokens=17, temperature=0.9, seed=3)
        a, b = (eng.requests[eng.add_request(q, s)] for q, s in ((p[0], sampling), (p[1], _sampling(max_tokens=60, logit_bias=((42, 100.0),)))))
        while a.request_id in eng.requests:
            assert ex.stats["rounds"] == 0
            eng.step()
        assert len(b.output) == len(a.output) >= 16
        if other == "grammar":
            assert a.output[-1] == eos and "".join(chr(t - 100) for t in a.output[:-1]) in options
        steps = eng.steps
        while eng.has_unfinished:
            eng.step()
        assert ex.stats["rounds"] > 0 and b.output == [42] * 60 and eng.steps - steps < 60 - len(a.output)
        runner.ws.check_status()
