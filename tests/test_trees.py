"""Drafts in trees and what requests say about their tokens: the host's part, and what the operators refuse before anything reaches a GPU."""
import numpy as np
import pytest
import torch

from cubic_serve_b200.ops import kernels as K
from cubic_serve_b200.runtime.trees import merge_drafts, tree_depths, tree_masks

I32 = torch.int32


def _ints(n, v=1):
    return torch.full((n,), v, dtype=I32)


def test_masks_and_depths_of_a_tree():
    parents = [-1, 0, 0, 1, 1, 2, 5]
    seen = [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 4}, {0, 2, 5}, {0, 2, 5, 6}]
    m = tree_masks(parents)
    assert m.shape == (7, 1) and m.dtype == np.uint32
    assert [{j for j in range(32) if r[0] >> np.uint32(j) & 1} for r in m] == seen
    assert tree_depths(parents).tolist() == [len(s) - 1 for s in seen]
    chain = tree_masks(list(range(-1, 69)))
    assert chain.shape == (70, 3) and all(sum(int(w).bit_count() for w in r) == j + 1 for j, r in enumerate(chain))
    assert tree_masks([-1], words=4).shape == (1, 4)


@pytest.mark.parametrize("parents,words", [([-1, 1], None), ([-1, 0, 2], None), ([-1, -1], None), (list(range(-1, 40)), 1)])
def test_masks_of_what_is_no_tree(parents, words):
    with pytest.raises(ValueError):
        tree_masks(parents, words)


def test_drafts_meet_in_a_tree():
    tokens, parents = merge_drafts([[5, 6, 7], [5, 8], [9], [5, 6, 7, 1]], 16)
    assert tokens == [0, 5, 6, 7, 8, 9, 1] and parents == [-1, 0, 1, 2, 1, 0, 3]
    assert merge_drafts([[5, 6, 7], [5, 8], [9]], 4) == ([0, 5, 6, 7, 8], [-1, 0, 1, 2, 1])
    assert merge_drafts([], 4) == ([0], [-1]) and merge_drafts([[1, 2]], 0) == ([0], [-1])


def _tree_args(**kw):
    a = dict(q=torch.zeros(6, 512, dtype=torch.bfloat16), out=torch.zeros(6, 512, dtype=torch.bfloat16), cache=torch.zeros(4, 2, K.kv_blob_bytes(128, 8, 8), dtype=torch.uint8),
             page_table=torch.zeros(3, 2, dtype=I32), request=_ints(2), row0=_ints(2), count=_ints(2), start=_ints(2), masks=torch.zeros(6, 1, dtype=I32), hq=4, hkv=2, head_dim=128,
             k_bits=8, v_bits=8, ws=K.Workspace(torch.device("cpu"), 16, 16, 16))
    a.update(kw)
    return a


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(6, 512)), dict(q=torch.zeros(6, 256, dtype=torch.bfloat16)), dict(out=torch.zeros(5, 512, dtype=torch.bfloat16)), dict(hq=3), dict(head_dim=64), dict(k_bits=5),
    dict(cache=torch.zeros(4, 2, 100, dtype=torch.uint8)), dict(cache=torch.zeros(4, 4, K.kv_blob_bytes(128, 8, 8), dtype=torch.uint8)[:, ::2]), dict(page_table=torch.zeros(3, 2)),
    dict(page_table=torch.zeros(3, 4, dtype=I32)[:, ::2]), dict(request=torch.ones(2)), dict(row0=_ints(1)), dict(count=_ints(4)[::2]), dict(start=torch.ones(2, dtype=torch.int64)),
    dict(masks=torch.zeros(5, 1, dtype=I32)), dict(masks=torch.zeros(6, 9, dtype=I32)), dict(masks=torch.zeros(6, 0, dtype=I32)), dict(masks=torch.zeros(6, 1, dtype=torch.int64)),
    dict(masks=torch.zeros(1, 1, dtype=I32).expand(6, 1)[:, :1].expand(6, 2)), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(hq=258, hkv=1),
    dict(q=torch.zeros(6, 516, dtype=torch.bfloat16)[:, :512]), dict(q=torch.zeros(6 * 512 + 4, dtype=torch.bfloat16)[4:].view(6, 512)), dict(request=_ints(1025), row0=_ints(1025)), dict(),
])
def test_tree_attention_refuses(change):
    with pytest.raises(ValueError):
        K.tree_attention(**_tree_args(**change))


def _adjust_args(**kw):
    a = dict(logits=torch.zeros(4, 100), request=_ints(4), history=torch.zeros(2, 10, dtype=I32), length=_ints(2), prompt=_ints(2), repetition=torch.ones(2), frequency=torch.ones(2),
             presence=torch.ones(2), bias=(_ints(3), _ints(5), torch.ones(5)), mask=torch.zeros(4, 4, dtype=I32), drafts=(_ints(4), torch.zeros(4, 1, dtype=I32), _ints(2)))
    a.update(kw)
    return a


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros(4, 100, dtype=torch.float16)), dict(logits=torch.zeros(4, 200)[:, ::2]), dict(logits=torch.zeros(1, 100).expand(4, 100)), dict(out=torch.zeros(4, 99)),
    dict(out=torch.zeros(4, 100, dtype=torch.bfloat16)), dict(request=_ints(3)), dict(request=None), dict(history=torch.zeros(2, 10)), dict(length=_ints(1)), dict(prompt=_ints(1)),
    dict(repetition=torch.ones(1)), dict(frequency=torch.ones(2, dtype=torch.float64)), dict(presence=torch.ones(4)[::2]), dict(bias=(_ints(2), _ints(5), torch.ones(5))),
    dict(bias=(_ints(3), _ints(5), torch.ones(4))), dict(mask=torch.zeros(3, 4, dtype=I32)), dict(mask=torch.zeros(4, 3, dtype=I32)), dict(mask=torch.zeros(4, 4)),
    dict(drafts=(_ints(3), torch.zeros(4, 1, dtype=I32), _ints(2))), dict(drafts=(_ints(4), torch.zeros(3, 1, dtype=I32), _ints(2))), dict(drafts=(_ints(4), torch.zeros(4, 9, dtype=I32), _ints(2))),
    dict(drafts=(_ints(4), torch.zeros(4, 1, dtype=I32), _ints(1))), dict(),
])
def test_adjust_logits_refuses(change):
    with pytest.raises(ValueError):
        K.adjust_logits(**_adjust_args(**change))


@pytest.mark.parametrize("logits,out,fits", [
    ((0, 100, 100), (400, 100, 100), True), ((400, 100, 100), (0, 100, 100), True), ((0, 100, 100), (0, 100, 100), True),        # beside, and the same
    ((0, 100, 100), (399, 100, 100), False), ((399, 100, 100), (0, 100, 100), False), ((0, 100, 100), (8, 100, 100), False), ((8, 100, 100), (0, 100, 100), False),
    ((0, 200, 100), (100, 200, 100), True), ((100, 200, 100), (0, 200, 100), True), ((0, 200, 100), (99, 200, 100), False), ((0, 200, 100), (101, 200, 100), False),
    ((0, 200, 100), (300, 200, 100), True), ((0, 208, 100), (104, 208, 100), True), ((0, 200, 100), (0, 100, 100), False), ((0, 100, 100), (0, 200, 100), False),
])
def test_results_of_adjusted_logits_beside_them_or_in_place(logits, out, fits):
    """``(first element, row stride, columns)`` of four rows of one buffer; what is accepted reaches the next check, which refuses for the GPU's sake."""
    buffer = torch.zeros(1200)
    a, b = (buffer[at:].as_strided((4, cols), (ld, 1), at) for at, ld, cols in (logits, out))
    with pytest.raises(ValueError) as e:
        K.adjust_logits(**_adjust_args(logits=a, out=b))
    assert ("apart" in str(e.value)) != fits


@pytest.mark.parametrize("change", [
    dict(tokens=_ints(5)), dict(parents=torch.ones(6)), dict(row0=torch.ones(2)), dict(count=_ints(1)), dict(accepted=_ints(1)), dict(path=torch.zeros(1, 4, dtype=I32)),
    dict(path=torch.zeros(2, 3, dtype=I32)), dict(path=torch.zeros(2, 8, dtype=I32)[:, ::2]), dict(emitted=torch.zeros(2, 4)), dict(path=torch.zeros(2, 0, dtype=I32), emitted=torch.zeros(2, 0, dtype=I32)), dict(),
])
def test_verify_tree_refuses(change):
    a = dict(target_ids=_ints(6), tokens=_ints(6), parents=_ints(6), row0=_ints(2), count=_ints(2), accepted=_ints(2), path=torch.zeros(2, 4, dtype=I32), emitted=torch.zeros(2, 4, dtype=I32))
    a.update(change)
    with pytest.raises(ValueError):
        K.verify_tree(**a)


def _caches(shapes, **kw):
    a = dict(hkv=2, head_dim=128, k_bits=8, v_bits=8)
    a.update(kw)
    return K.LayerCaches([torch.zeros(*s, dtype=torch.uint8) for s in shapes], **a)


@pytest.mark.parametrize("shapes,kw", [([(4, 2, 4608), (5, 2, 4608)], {}), ([(4, 2, 4608)], dict(hkv=1)), ([(4, 2, 4608)], dict(k_bits=4)), ([(4, 2, 4608)], dict(v_bits=7)),
                                       ([(4, 2, 4608)], dict(head_dim=64)), ([(0, 2, 4608)], {}), ([], {})])
def test_layer_caches_refuse(shapes, kw):
    with pytest.raises(ValueError):
        _caches(shapes, **kw)


@pytest.mark.parametrize("change", [
    dict(page_table=torch.zeros(3, 2)), dict(request=torch.ones(2)), dict(start=_ints(1)), dict(accepted=_ints(1)), dict(path=torch.zeros(1, 4, dtype=I32)), dict(path=torch.zeros(2, 4)), dict(),
])
def test_keep_tokens_refuses(change):
    caches = _caches([(4, 2, 4608), (0, 2, 4608), (4, 2, 4608)])
    assert len(caches.caches) == 2
    a = dict(caches=caches, page_table=torch.zeros(3, 2, dtype=I32), request=_ints(2), start=_ints(2), accepted=_ints(2), path=torch.zeros(2, 4, dtype=I32),
             ws=K.Workspace(torch.device("cpu"), 16, 16, 16))
    a.update(change)
    with pytest.raises(ValueError):
        K.keep_tokens(**a)


# ------------------------------------------------------------------------------------------------- what requests say
def test_requests_say_what_their_logits_are():
    from cubic_serve_b200.contracts.request import RequestError
    from cubic_serve_b200.inputs.normalize import normalize_openai_chat_completions
    body = {"model": "m", "messages": [{"role": "user", "content": "hi"}]}
    s = normalize_openai_chat_completions({**body, "repetition_penalty": 1.2, "presence_penalty": 0.5, "logit_bias": {"17": -100, "4": 2.5}}).sampling
    assert (s.repetition_penalty, s.presence_penalty, s.logit_bias) == (1.2, 0.5, ((17, -100.0), (4, 2.5)))
    s = normalize_openai_chat_completions(body).sampling
    assert (s.repetition_penalty, s.logit_bias) == (1.0, ())
    for bad in ({"repetition_penalty": 0}, {"repetition_penalty": -1}, {"logit_bias": [1]}, {"logit_bias": {"a": 1}}, {"logit_bias": {"-3": 1}}, {"logit_bias": {"3": "1"}},
                {"logit_bias": {"3": 101}}, {"logit_bias": {str(i): 0 for i in range(1025)}}, {"logit_bias": {"3": float("nan")}}):
        with pytest.raises(RequestError):
            normalize_openai_chat_completions({**body, **bad})


@pytest.mark.parametrize("bad", [{"logit_bias": {"3": 10 ** 400}}, {"logit_bias": {"3": -10 ** 400}}, {"logit_bias": {"9" * 5000: 1}},
                                 {"repetition_penalty": 10 ** 400}])
def test_numbers_of_any_length_are_requests_errors(bad):
    """Whole numbers in JSON may be longer than what Python turns into a float, or a text into a number."""
    from cubic_serve_b200.contracts.request import RequestError
    from cubic_serve_b200.inputs.normalize import normalize_openai_chat_completions
    with pytest.raises(RequestError):
        normalize_openai_chat_completions({"model": "m", "messages": [{"role": "user", "content": "hi"}], **bad})


def test_sampling_parameters_of_adjustments():
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    assert not SamplingParams().adjusts and SamplingParams(presence_penalty=0.1).adjusts and SamplingParams(logit_bias=((1, 2.0),)).adjusts
    for bad in (dict(repetition_penalty=0.0), dict(frequency_penalty=2.5), dict(presence_penalty=-3.0), dict(logit_bias=((-1, 0.0),)), dict(logit_bias=((1, 101.0),)),
                dict(logit_bias=tuple((i, 0.0) for i in range(1025)))):
        with pytest.raises(ValueError):
            SamplingParams(**bad).validate()


def test_histories_are_staged_as_they_grow():
    from types import SimpleNamespace as S

    from cubic_serve_b200.executor.adjustments import Adjustment, Adjustments
    a = Adjustments(4, 10, "cpu")
    tokens = [5, 6, 7]
    seg = S(request_slot=2, uid=9, adjust=Adjustment(tokens, 2, 1.5, 0.5, 0.25, ((3, 1.0), (8, -2.0))))
    none = S(request_slot=1, uid=4, adjust=None)
    d = a.stage([none, seg])
    assert d["request"].tolist() == [-1, 2] and d["length"].tolist() == [0, 0, 3, 0] and d["prompt"].tolist() == [0, 0, 2, 0]
    assert d["history"][2, :3].tolist() == tokens and d["repetition"].tolist() == [1.0, 1.0, 1.5, 1.0] and d["presence"][2].item() == 0.25
    assert d["bias"][0].tolist() == [0, 0, 0, 2, 2] and d["bias"][1].tolist() == [3, 8] and d["bias"][2].tolist() == [1.0, -2.0]
    tokens += [8, 9]
    assert a.stage([seg], [3])["request"].tolist() == [2, 2, 2] and a.history[2, :5].tolist() == tokens
    other = S(request_slot=2, uid=10, adjust=Adjustment([1], 1))                              # another request in the slot
    d = a.stage([other])
    assert d["length"][2].item() == 1 and a.history[2, 0].item() == 1 and "bias" not in d
    long = S(request_slot=0, uid=11, adjust=Adjustment(list(range(14)), 12))                  # longer than there is room for
    assert a.stage([long])["length"][0].item() == 10


def test_several_continuations_of_a_history():
    from cubic_serve_b200.runtime.ngram import NgramIndex, NgramProposer
    x = NgramIndex(3, 1, 4)
    x.extend([1, 2, 3, 1, 2, 4, 1, 2, 5, 1, 2])
    assert x.propose(2) == [5, 1] and x.propose_many(2) == [[5, 1], [4, 1], [3, 1]] and x.propose_many(0) == []
    y = NgramIndex(3, 1, 2)
    y.extend([1, 2, 3, 1, 2, 4, 1, 2, 5, 1, 2])
    assert y.propose_many(3) == [[5, 1, 2], [4, 1, 2]]
    p = NgramProposer(positions=3)
    assert p.propose_many("a", [1, 2, 9, 1, 2], 2) == [[9, 1]] and p.propose("a", [1, 2, 9, 1, 2], 2) == [9, 1]
    with pytest.raises(ValueError):
        NgramIndex(positions=0)


def test_branches_on_the_command_line():
    import argparse

    from cubic_serve_b200.cli import parse_speculative_config
    assert parse_speculative_config('{"method":"ngram","num_speculative_tokens":4,"branches":3}').branches == 3
    assert parse_speculative_config('{"method":"ngram","num_speculative_tokens":4}').branches == 1
    for bad in ('{"method":"ngram","num_speculative_tokens":4,"branches":0}', '{"method":"ngram","num_speculative_tokens":4,"branches":17}',
                '{"method":"ngram","num_speculative_tokens":4,"branches":true}', '{"method":"mtp","num_speculative_tokens":4,"branches":2}'):
        with pytest.raises(argparse.ArgumentTypeError):
            parse_speculative_config(bad)


def test_memory_of_what_requests_may_ask_for():
    from cubic_serve_b200.executor.adjustments import Adjustments
    from cubic_serve_b200.executor.gpu_executor import BatchBuilder
    from cubic_serve_b200.runtime.serving import request_buffers_bytes

    def histories(running, length):
        return Adjustments(running, 16 * BatchBuilder(running, 64, length, 4, 2, "cpu").max_pages, "cpu").history.nbytes
    assert request_buffers_bytes(8, 1000, 512, 2048) == histories(8, 1000)
    assert request_buffers_bytes(8, 1000, 512, 2048, 4) == 0                                  # chains of drafts: neither
    assert request_buffers_bytes(8, 1000, 512, 2048, 4, 4) == histories(8, 1017) + 2 * 2048 * 8 * 17
    assert request_buffers_bytes(256, 8192, 8192, 151936, 7, 16) == histories(256, 8305) + 2 * 151936 * 8192       # a pass of 8192 rows


class _TreeExecutor:
    """An executor of rounds with trees without a GPU: the target says 7 over and over, and so every draft of it is accepted."""
    draft_source, speculative_sampling, speculative_grammar = "ngram", False, False

    def __init__(self, depth, branches):
        self.draft_depth, self.draft_branches, self.speculative_depth = depth, branches, depth * branches
        self.rounds, self.forgotten = [], []

    def execute(self, segs):
        return [7 for s in segs if s.sample]

    def copy_pages(self, pairs):
        pass

    def invalidate_page_rows(self, slots):
        self.forgotten += list(slots)

    def execute_speculative(self, segs, depths=None, drafts=None):
        self.rounds.append([(len(s.pages), s.start, [list(c) for c in d]) for s, d in zip(segs, drafts)])
        out = []
        for s, d in zip(segs, drafts):
            tree = merge_drafts(d, max(0, len(s.pages) * 16 - s.start - 1))[0]
            n = 0
            while n < len(tree) - 1 and tree[n + 1] == 7:
                n += 1
            out.append([7] * (n + 1))
        return out


def _tree_engine(depth, branches, pages, requests=2, **kw):
    from cubic_serve_b200.runtime.engine import LLMEngine
    from cubic_serve_b200.runtime.scheduler import SchedulerConfig
    ex = _TreeExecutor(depth, branches)
    return LLMEngine(ex, pages, SchedulerConfig(max_running_requests=requests, max_model_len=512, max_batched_tokens=256, enable_prefix_cache=False)), ex


@pytest.mark.parametrize("branches", [1, 4])
def test_an_executor_of_trees_is_given_lists_of_continuations(branches):
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    eng, ex = _tree_engine(3, branches, 64)
    assert eng.generate([[7] * 9, [1, 2, 3]], SamplingParams(max_tokens=12, ignore_eos=True)) == [[7] * 12] * 2
    assert any(d == [[7, 7, 7]] for r in ex.rounds for _, _, d in r)


def test_drafts_in_trees_hold_pages_for_their_round_alone():
    """Requests without a match hold what plain ones do; those with one are lent pages for what they draft, and give them back."""
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    eng, ex = _tree_engine(7, 16, 64)
    a, b = (eng.add_request(p, SamplingParams(max_tokens=40, ignore_eos=True)) for p in ([1, 2, 3, 4], [7, 7, 1, 2, 3, 4, 5, 6, 7, 7, 11, 12, 13, 14, 15, 16, 7, 7, 21, 22, 23, 24, 25, 26]))
    a, b = eng.requests[a], eng.requests[b]
    while eng.has_unfinished:
        eng.step()
        for r in (a, b):
            assert len(r.pages) <= -(-(r.num_computed + 1) // 16)
        assert eng.pool.num_used == len(a.pages) + len(b.pages)
    assert a.output == b.output == [7] * 40
    drafted = [(pages, start, len(merge_drafts(d, 112)[0])) for r in ex.rounds for pages, start, d in r]
    assert {n > 1 for _, _, n in drafted} == {True, False}
    assert all(pages == -(-(start + n) // 16) for pages, start, n in drafted), "as many slots as the drafts can take"
    assert ex.forgotten, "rows of the block table whose pages were given back are written anew"


def test_drafts_in_trees_preempt_nobody():
    """Eight requests that repeat themselves in a pool that just holds their tokens: all drafts have less room, no request loses its place or its last tokens."""
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    eng, ex = _tree_engine(7, 16, 1 + 8 * 4, requests=8)
    reqs = [eng.requests[eng.add_request([7] * 9 + [i], SamplingParams(max_tokens=54, ignore_eos=True))] for i in range(8)]
    while eng.has_unfinished:
        eng.step()
    assert [r.preemptions for r in reqs] == [0] * 8 and [r.output for r in reqs] == [[7] * 54] * 8
    assert eng.steps < 54 and eng.pool.num_used == 0


def test_drafts_in_trees_shorten_no_request():
    """A request alone in a pool that its last token fills."""
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    eng, ex = _tree_engine(7, 16, 1 + 3)
    assert eng.generate([[7] * 9], SamplingParams(max_tokens=39, ignore_eos=True)) == [[7] * 39]


def test_tokens_that_could_not_be_staged_are_staged_by_the_next_step():
    from types import SimpleNamespace as S

    from cubic_serve_b200.executor.adjustments import Adjustment, Adjustments
    a = Adjustments(2, 10, "cpu")
    segs = [S(request_slot=0, uid=1, adjust=Adjustment([5, 6], 2)), S(request_slot=1, uid=2, adjust=Adjustment([7], 1, bias=((1 << 40, 1.0),)))]
    with pytest.raises(OverflowError):
        a.stage(segs)
    segs[0].adjust.tokens.append(9)
    assert a.stage(segs[:1])["length"].tolist() == [3, 0] and a.history[0, :3].tolist() == [5, 6, 9]


def test_an_executor_of_trees_without_a_block_table_of_its_own():
    """Executors need not keep rows of pages (``models/protocol.py``)."""
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    eng, ex = _tree_engine(7, 16, 64)
    plain = type("PlainRows", (), {k: getattr(ex, k) for k in ("draft_source", "speculative_sampling", "speculative_grammar", "draft_depth", "draft_branches", "speculative_depth", "execute",
                                                              "copy_pages", "execute_speculative")})()
    eng.executor = plain
    prompt = [7, 7, 1, 2, 3, 4, 5, 6, 7, 7, 11, 12, 13, 14, 15, 16, 7, 7, 21, 22, 23, 24, 25, 26]
    assert eng.generate([prompt], SamplingParams(max_tokens=20, ignore_eos=True)) == [[7] * 20]
