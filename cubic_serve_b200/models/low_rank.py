"""Low-rank adapters of a decoder: what requests may name, beside the weights that they share.

An adapter gives projections of a layer ``y + scale (x A^T) B^T``.  All adapters of a deployment live in slots of one bank a
projection (``ops.kernels.AdapterBank``), so a step's requests may each name their own; its rows are sorted by adapter once.
Adapters come as directories of ``adapter_config.json`` and ``adapter_model.safetensors`` (A and B of
``layers.N.self_attn.{q,k,v,o}_proj`` and ``layers.N.mlp.{gate,up,down}_proj``).
"""
from __future__ import annotations

import json
import math
import re
from dataclasses import dataclass
from pathlib import Path

import torch

from ..ops import kernels as K

#: section of a projection -> the module of a checkpoint that it is
SECTIONS = {"qkv": ("q_proj", "k_proj", "v_proj"), "o": ("o_proj",), "gate_up": ("gate_proj", "up_proj"), "down": ("down_proj",)}
_KEY = re.compile(r"(?:^|\.)layers\.(\d+)\.(?:self_attn|mlp)\.(\w+_proj)\.lora_([AB])\.weight$")


class AdapterError(ValueError):
    """An adapter that this deployment cannot serve, or a name that it does not know."""


@dataclass(frozen=True)
class LoadedAdapter:
    name: str
    slot: int
    #: differs between loads, so that pages of the prefix cache are never shared between adapters or versions of one
    key: bytes


def read_adapter(path) -> tuple[dict, float, int]:
    """``({(layer, module): (A, B)}, scale, rank)`` of an adapter directory."""
    path = Path(path)
    try:
        cfg = json.loads((path / "adapter_config.json").read_text())
    except (OSError, ValueError) as exc:
        raise AdapterError(f"{path}: no readable adapter_config.json: {exc}") from exc
    if not isinstance(cfg, dict):
        raise AdapterError(f"{path}: adapter_config.json is not an object")
    for field in ("use_dora", "modules_to_save", "rank_pattern", "alpha_pattern", "fan_in_fan_out", "lora_bias"):
        if cfg.get(field):
            raise AdapterError(f"{path}: adapters with {field} are not served")
    if cfg.get("bias", "none") != "none":
        raise AdapterError(f"{path}: adapters with biases are not served")
    rank, alpha = cfg.get("r"), cfg.get("lora_alpha")
    if not isinstance(rank, int) or isinstance(rank, bool) or rank < 1 or not isinstance(alpha, (int, float)) or isinstance(alpha, bool) or not math.isfinite(alpha):
        raise AdapterError(f"{path}: r and lora_alpha must be numbers, r at least 1")
    try:
        from safetensors.torch import load_file
        tensors = load_file(str(path / "adapter_model.safetensors"))
    except Exception as exc:  # noqa: BLE001 - whatever the reader met, the adapter is not served
        raise AdapterError(f"{path}: no readable adapter_model.safetensors: {exc}") from exc
    found: dict[tuple[int, str], dict] = {}
    for key, t in tensors.items():
        m = _KEY.search(key)
        if m is None or t.dim() != 2:
            raise AdapterError(f"{path}: {key} is not a matrix of a projection that adapters may change")
        found.setdefault((int(m[1]), m[2]), {})[m[3]] = t
    for (layer, module), ab in found.items():
        if set(ab) != {"A", "B"} or ab["A"].shape[0] != rank or ab["B"].shape[1] != rank:
            raise AdapterError(f"{path}: layer {layer} {module}: A [{rank}, in] and B [out, {rank}] are wanted")
    if not found:
        raise AdapterError(f"{path}: no matrices")
    return {k: (v["A"], v["B"]) for k, v in found.items()}, alpha / (math.sqrt(rank) if cfg.get("use_rslora") else rank), rank


class LowRankAdapters:
    """The banks of a decoder's projections, and the sorted rows of its steps."""

    def __init__(self, cfg, layers: list, slots: int, max_rank: int, max_tokens: int, device) -> None:
        """``layers``: the decoder's ``LayerWeights``.  Full-attention layers take adapters on q, k, v and o, dense MLPs on gate, up and
        down; experts and recurrent mixers have none.  ``nbytes``: memory that all of it holds (a server plans with that of one on
        the device ``meta``)."""
        if not 1 <= slots <= 1023 or not 1 <= max_rank <= 128:
            raise AdapterError("up to 1023 adapters of ranks up to 128")
        self.slots, self.max_rank = slots, max_rank
        D = cfg.head_dim
        q, kv, h, i = cfg.num_q_heads * D, cfg.num_kv_heads * D, cfg.hidden_size, cfg.intermediate_size
        shapes = {"qkv": (h, (q, kv, kv)), "o": (q, (h,)), "gate_up": (h, (i, i)), "down": (i, (h,))}
        self.banks: list[dict[str, K.AdapterBank]] = []
        most = 0
        for lw in layers:
            names = ([] if lw.gdn is not None else ["qkv", "o"]) + ([] if lw.moe is not None else ["gate_up", "down"])
            banks = {}
            for name in names:
                k, widths = shapes[name]
                zero = torch.zeros((), dtype=torch.bfloat16, device=device)
                banks[name] = K.AdapterBank(zero.expand(slots, len(widths) * max_rank, k), zero.expand(slots, sum(widths), max_rank),
                                            torch.zeros(slots, device=device), widths, ranks=torch.zeros(slots, dtype=torch.int32, device=device))
                most = max(most, len(widths) * max_rank)
            self.banks.append(banks)
        self.rows = K.AdapterRows(max_tokens, slots, max(most, 1), device)
        self.nbytes = self.rows.nbytes + sum(bank.nbytes for banks in self.banks for bank in banks.values())
        self.loaded: dict[str, LoadedAdapter] = {}
        self._loads = 0

    def load(self, name: str, path) -> LoadedAdapter:
        """Put the adapter of a directory into a free slot.  Requests that decode meanwhile are not disturbed: no row names the slot."""
        if not name or name in self.loaded:
            raise AdapterError(f"an adapter named {name!r} is loaded already" if name else "an adapter needs a name")
        free = set(range(self.slots)) - {a.slot for a in self.loaded.values()}
        if not free:
            raise AdapterError(f"all {self.slots} slots hold adapters")
        matrices, scale, rank = read_adapter(path)
        if rank > self.max_rank:
            raise AdapterError(f"{path}: rank {rank}; this deployment keeps ranks up to {self.max_rank}")
        slot, left = min(free), dict(matrices)
        try:
            for li, banks in enumerate(self.banks):
                for proj, bank in banks.items():
                    ab = [left.pop((li, module), (None, None)) for module in SECTIONS[proj]]
                    bank.load(slot, [a for a, _ in ab], [b for _, b in ab], scale)
        except ValueError as exc:
            self._clear(slot)
            raise AdapterError(f"{path}: layer {li} {proj}: {exc}") from exc
        if left:
            self._clear(slot)
            raise AdapterError(f"{path}: layer {min(left)[0]} {min(left)[1]} takes no adapter in this model")
        self._loads += 1
        got = self.loaded[name] = LoadedAdapter(name, slot, f"{self._loads}:{name}".encode())
        return got

    def unload(self, name: str) -> None:
        """Free an adapter's slot; no request may still name it."""
        self._clear(self.get(name).slot)
        del self.loaded[name]

    def _clear(self, slot: int) -> None:
        for banks in self.banks:
            for bank in banks.values():
                bank.load(slot, [None] * bank.sections, [None] * bank.sections, 0.0)

    def get(self, name: str) -> LoadedAdapter:
        if name not in self.loaded:
            raise AdapterError(f"no adapter named {name!r} is loaded")
        return self.loaded[name]

    # ------------------------------------------------------------------ steps
    def begin(self, row_slots: torch.Tensor) -> None:
        """Sort the rows of the step that follows: int32, the adapter slot of every row (-1: none)."""
        K.adapter_rows(row_slots, self.rows)

    def add(self, layer: int, proj: str, x: torch.Tensor, y: torch.Tensor) -> int:
        """Add the adapters' part of a projection to its result ``y``, in place; returns the launches."""
        bank = self.banks[layer].get(proj)
        if bank is None:
            return 0
        K.adapter_add(x, y, bank, self.rows)
        return 1 if self.rows.rows <= K.ADAPTER_FEW_ROWS else 2
