"""Low-rank adapters and whole-vocabulary draws off the GPU: files, names, refusals, wire fields, the eager draw."""
import json

import numpy as np
import pytest
import torch

from cubic_serve_b200.models.config import ModelConfig, QuantSpec
from cubic_serve_b200.models.low_rank import AdapterError, LowRankAdapters, read_adapter

CFG = ModelConfig(name="t", num_layers=2, hidden_size=64, num_q_heads=2, num_kv_heads=1, head_dim=32, intermediate_size=96, vocab_size=128, quant=QuantSpec("none"))
SHAPES = {"self_attn.q_proj": (64, 64), "self_attn.k_proj": (32, 64), "self_attn.v_proj": (32, 64), "self_attn.o_proj": (64, 64), "mlp.gate_proj": (96, 64), "mlp.up_proj": (96, 64),
          "mlp.down_proj": (64, 96)}


class _Layer:
    gdn = moe = None


def _write(path, names=tuple(SHAPES), rank=4, layers=(0, 1), extra=None, **cfg):
    from safetensors.torch import save_file
    path.mkdir(exist_ok=True)
    t = {}
    for i in layers:
        for n in names:
            out, k = SHAPES[n]
            t[f"base_model.model.model.layers.{i}.{n}.lora_A.weight"] = torch.randn(rank, k)
            t[f"base_model.model.model.layers.{i}.{n}.lora_B.weight"] = torch.randn(out, rank)
    t.update(extra or {})
    save_file(t, str(path / "adapter_model.safetensors"))
    (path / "adapter_config.json").write_text(json.dumps({"r": rank, "lora_alpha": 8, **cfg}))
    return t


def test_adapters_are_read_and_take_slots(tmp_path):
    t = _write(tmp_path / "a")
    _write(tmp_path / "b", names=("self_attn.v_proj",), rank=2, layers=(1,), use_rslora=True)
    m, scale, rank = read_adapter(tmp_path / "a")
    assert scale == 2.0 and rank == 4 and len(m) == 14 and torch.equal(m[1, "k_proj"][0], t["base_model.model.model.layers.1.self_attn.k_proj.lora_A.weight"])
    assert read_adapter(tmp_path / "b")[1] == pytest.approx(8 / 2 ** 0.5)
    lr = LowRankAdapters(CFG, [_Layer(), _Layer()], 2, 8, 16, "cpu")
    a, b = lr.load("a", tmp_path / "a"), lr.load("b", tmp_path / "b")
    assert (a.slot, b.slot) == (0, 1) and a.key != b.key
    qkv = lr.banks[1]["qkv"]
    got = qkv.a.transpose(1, 2).reshape(2, 3, 16, 64)
    assert torch.equal(got[0, 1, :4], t["base_model.model.model.layers.1.self_attn.k_proj.lora_A.weight"].bfloat16()) and not got[:, :, 4:].any() and not got[1, :2].any()
    assert qkv.ranks.tolist() == [4, 2] and lr.banks[0]["qkv"].ranks.tolist() == [4, 0] and lr.banks[1]["down"].ranks.tolist() == [4, 0]
    with pytest.raises(AdapterError):
        lr.load("c", tmp_path / "a")
    lr.unload("a")
    assert not got.new_tensor(lr.banks[0]["qkv"].ranks.tolist()).any() and not lr.banks[0]["o"].a[0].any()
    c = lr.load("a", tmp_path / "a")
    assert c.slot == 0 and c.key != a.key, "what was cached with the earlier load is not taken for the later one's"
    with pytest.raises(AdapterError):
        lr.get("d")


@pytest.mark.parametrize("change", [
    dict(use_dora=True), dict(bias="all"), dict(modules_to_save=["lm_head"]), dict(rank_pattern={"q": 2}), dict(r=0), dict(r="4"), dict(lora_alpha=None), dict(lora_alpha=float("nan")), dict(r=5),
])
def test_adapter_configs_that_are_not_served(tmp_path, change):
    _write(tmp_path / "a", **{k: v for k, v in change.items() if k not in ("r", "lora_alpha")})
    cfg = json.loads((tmp_path / "a" / "adapter_config.json").read_text())
    (tmp_path / "a" / "adapter_config.json").write_text(json.dumps({**cfg, **change}))
    with pytest.raises(AdapterError):
        read_adapter(tmp_path / "a")


def test_adapter_files_that_are_not_served(tmp_path):
    with pytest.raises(AdapterError):
        read_adapter(tmp_path / "none")
    _write(tmp_path / "a", extra={"base_model.model.lm_head.lora_A.weight": torch.zeros(4, 64)})
    with pytest.raises(AdapterError):
        read_adapter(tmp_path / "a")
    _write(tmp_path / "b", extra={"base_model.model.model.layers.0.mlp.up_proj.lora_A.weight": torch.zeros(3, 64)})
    with pytest.raises(AdapterError):
        read_adapter(tmp_path / "b")
    lr = LowRankAdapters(CFG, [_Layer(), _Layer()], 1, 8, 16, "cpu")
    _write(tmp_path / "c", layers=(0, 1, 2))
    _write(tmp_path / "d", extra={"base_model.model.model.layers.0.mlp.up_proj.lora_B.weight": torch.zeros(90, 4)})
    for name in "cd":
        with pytest.raises(AdapterError):
            lr.load(name, tmp_path / name)
        assert not lr.loaded and not any(bank.a.any() or bank.ranks.any() for banks in lr.banks for bank in banks.values()), "nothing of it stays"
    moe = _Layer()
    moe.moe = object()
    with pytest.raises(AdapterError):
        LowRankAdapters(CFG, [moe, _Layer()], 1, 8, 16, "cpu").load("a", _write(tmp_path / "e") and tmp_path / "e")


def test_command_line_of_adapters():
    from types import SimpleNamespace

    from cubic_serve_b200.runtime.serving import _low_rank_adapters
    ns = lambda *a, slots=None: SimpleNamespace(low_rank_adapter=list(a), low_rank_slots=slots, low_rank_max_rank=32)        # noqa: E731
    assert _low_rank_adapters(ns()) is None and _low_rank_adapters(ns("x=/d=1", "y=e")) == ((2, 32), [("x", "/d=1"), ("y", "e")])
    assert _low_rank_adapters(ns(slots=4)) == ((4, 32), [])
    for bad in (ns("x"), ns("=d"), ns("x=d", "x=e"), ns("x=d", "y=e", slots=1)):
        with pytest.raises(SystemExit):
            _low_rank_adapters(bad)


def test_wire_fields_of_whole_vocabulary_draws():
    from cubic_serve_b200.contracts.request import RequestError
    from cubic_serve_b200.inputs.normalize import normalize_openai_chat_completions as n
    body = {"model": "m", "messages": [{"role": "user", "content": "x"}]}
    s = n({**body, "whole_vocabulary": True, "top_k": 500}, "m").sampling
    assert s.whole_vocabulary and s.top_k == 500 and s.min_p == 0.0
    assert n({**body, "min_p": 0.1, "top_k": 40}, "m").sampling.min_p == 0.1 and not n(body, "m").sampling.whole_vocabulary
    for bad in ({"top_k": 21}, {"min_p": -0.1}, {"min_p": 1.5}, {"whole_vocabulary": 1}, {"whole_vocabulary": True, "top_k": -1}, {"min_p": "a"}):
        with pytest.raises(RequestError):
            n({**body, **bad}, "m")
    from cubic_serve_b200.runtime.scheduler import SamplingParams
    SamplingParams(top_k=500, whole_vocabulary=True).validate()
    for bad in (dict(top_k=21), dict(min_p=2.0), dict(top_k=2 ** 31, min_p=0.1)):
        with pytest.raises(ValueError):
            SamplingParams(**bad).validate()


def test_the_eager_draw_keeps_prefixes():
    from cubic_serve_b200.executor.eager_executor import sample_row
    from cubic_serve_b200.executor.gpu_executor import Segment
    logits = torch.tensor([0.0, 3.0, 3.0, -1.0, 2.0, float("-inf"), float("nan")])
    draw = lambda **kw: {sample_row(logits, Segment(0, [1], 0, [0], seed=i, whole=True, **{"temperature": 1.0, **kw})) for i in range(300)}        # noqa: E731
    assert draw() == {0, 1, 2, 3, 4} and draw(top_k=1) == {1} and draw(top_k=2) == {1, 2} and draw(min_p=0.3) == {1, 2, 4} and draw(top_p=0.5) == {1, 2}
    assert draw(temperature=50.0, top_k=30) == {0, 1, 2, 3, 4} and draw(min_p=1.0) == {1, 2}
    mask = np.array([0b11000], dtype=np.uint32)
    assert draw(mask=mask) == {3, 4}


def test_requests_name_adapters_as_models():
    import asyncio

    from cubic_serve_b200.api.server import CubicASGIApp

    class Backend:
        ready, adapter_names, seen = True, ("legal",), None

        def start(self, req):
            self.seen = req.model
            raise __import__("cubic_serve_b200.contracts.request", fromlist=["RequestError"]).RequestError("stop here", param="model", status=418)

    def call(path, method="GET", body=None):
        out = []

        async def receive():
            return {"type": "http.request", "body": json.dumps(body).encode() if body else b"", "more_body": False}

        async def send(m):
            out.append(m)
        asyncio.run(app({"type": "http", "method": method, "path": path, "headers": [(b"content-type", b"application/json")]}, receive, send))
        return out[0]["status"], b"".join(m.get("body", b"") for m in out)

    backend = Backend()
    app = CubicASGIApp(backend, "base", ["public", "other"])
    ask = lambda model: call("/v1/chat/completions", "POST", {"model": model, "messages": [{"role": "user", "content": "x"}]})        # noqa: E731
    assert [d["id"] for d in json.loads(call("/v1/models")[1])["data"]] == ["public", "legal"]
    for model, seen in (("legal", "legal"), ("other", "public"), ("base", "public")):
        assert ask(model)[0] == 418 and backend.seen == seen
    assert ask("unknown")[0] == 404


def test_a_name_of_the_model_reaches_no_adapter():
    from types import SimpleNamespace

    from cubic_serve_b200.api.server import CubicASGIApp
    from cubic_serve_b200.runtime.async_engine import TokenChatBackend
    backend = TokenChatBackend.__new__(TokenChatBackend)              # without its thread
    backend.engine, backend.model_names = SimpleNamespace(adapter_names=("public", "legal", "base")), frozenset()
    assert backend.adapter_names == ("public", "legal", "base")
    CubicASGIApp(backend, "base", ["public", "other"])
    assert backend.adapter_names == ("legal",)
