"""What requests say about their logits, on the device: token histories by request slot, penalties and biases (``K.adjust_logits``)."""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch


@dataclass
class Adjustment:
    """Penalties and biases of one request (``runtime.scheduler.SamplingParams``), and the tokens that they look at."""
    tokens: list[int]            # prompt and output so far
    prompt: int                  # how many of them are the prompt's
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: tuple[tuple[int, float], ...] = ()


class Adjustments:
    """Histories ``[slots, most]`` that grow with their requests: a step uploads the tokens that are new and a few numbers a slot, in
    one copy.  ``stage`` is called on the stream of the steps, when that stream has left the copy of the call before; what it
    returns holds until the next call."""

    def __init__(self, slots: int, most: int, device) -> None:
        self.slots, self.most, self.device = slots, most, torch.device(device)
        self.history = torch.zeros(slots, most, dtype=torch.int32, device=device)
        self._have: list[tuple[int, int]] = [(-2, 0)] * slots          # whose tokens a row holds, and how many
        self._host = self._dev = torch.empty(0, dtype=torch.uint8)

    def _upload(self, arrays: dict) -> dict:
        """The arrays on the device, by way of one pinned buffer and one copy."""
        at, end = {}, 0
        for name, a in arrays.items():
            at[name], end = end, end + -(-a.nbytes // 16) * 16
        if end > self._host.numel():
            size = max(end, 2 * self._host.numel(), 1 << 16)
            self._host = torch.empty(size, dtype=torch.uint8, pin_memory=self.device.type == "cuda")
            self._dev = torch.empty(size, dtype=torch.uint8, device=self.device)
        h, out = self._host.numpy(), {}
        for name, a in arrays.items():
            h[at[name]:at[name] + a.nbytes] = np.ascontiguousarray(a).reshape(-1).view(np.uint8)
        self._dev[:end].copy_(self._host[:end], non_blocking=True)
        for name, a in arrays.items():
            out[name] = self._dev[at[name]:at[name] + a.nbytes].view(getattr(torch, a.dtype.name)).view(a.shape)
        return out

    def stage(self, segs, rows: list[int] | None = None) -> dict:
        """Operands of ``K.adjust_logits`` for one row of logits a segment, or ``rows[i]`` neighbouring rows of segment i."""
        n = self.slots
        ints = np.zeros((2, n), dtype=np.int32)                        # length, prompt
        floats = np.zeros((3, n), dtype=np.float32)                    # repetition, frequency, presence
        floats[0] = 1.0
        where, what, bias, held = [], [], {}, {}
        for s in segs:
            a = s.adjust
            if a is None:
                continue
            slot, L = s.request_slot, min(len(a.tokens), self.most)
            uid, have = self._have[slot]
            if uid != s.uid or s.uid < 0 or have > L:
                have = 0
            where.append(np.arange(slot * self.most + have, slot * self.most + L, dtype=np.int64))
            what.append(np.asarray(a.tokens[have:L], dtype=np.int32))
            held[slot] = (s.uid, L)
            ints[:, slot] = L, min(a.prompt, L)
            floats[:, slot] = a.repetition, a.frequency, a.presence
            if a.bias:
                bias[slot] = a.bias
        request = np.repeat(np.array([s.request_slot if s.adjust is not None else -1 for s in segs], dtype=np.int32), rows or [1] * len(segs))
        arrays = {"where": np.concatenate(where) if where else np.zeros(0, dtype=np.int64), "what": np.concatenate(what) if what else np.zeros(0, dtype=np.int32),
                  "ints": ints, "floats": floats, "request": request}
        if bias:
            count = np.zeros(n + 1, dtype=np.int32)
            for slot, b in bias.items():
                count[slot + 1] = len(b)
            pairs = [p for slot in sorted(bias) for p in bias[slot]]
            arrays.update(first=np.cumsum(count, dtype=np.int32), ids=np.array([t for t, _ in pairs], dtype=np.int32), values=np.array([v for _, v in pairs], dtype=np.float32))
        d = self._upload(arrays)
        if d["where"].numel():
            self.history.view(-1).index_copy_(0, d["where"], d["what"])
        for slot, have in held.items():          # (once the tokens are on their way: not if anything above failed)
            self._have[slot] = have
        out = dict(request=d["request"], history=self.history, length=d["ints"][0], prompt=d["ints"][1], repetition=d["floats"][0], frequency=d["floats"][1],
                   presence=d["floats"][2])
        if bias:
            out["bias"] = (d["first"], d["ids"], d["values"])
        return out
