"""What a step does for each of its requests: where its tokens go, which adapter its rows take, how its next token is drawn.

Three operators that a step of a server runs around the shared layers.

* The step's layout: from the requests' lengths, their new tokens and the pages they are given, the block table, the slot and
  the position of every token and the row blocks of the attention.
* Low-rank adapters of many requests beside a shared projection: ``y + scale (x A^T) B^T`` with the A and B of each row's own
  adapter.  A pass is one decoder layer: the rows are sorted by adapter once, then the four projections of the layer follow.
* The draw from a whole vocabulary: temperature, top-k, top-p and min-p of each row, from a given uniform number.

The plain forms are elementary torch operations over all rows at once, in 32 bits, or in 64 where a sum over a vocabulary is
compared with a border.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16


# ------------------------------------------------------------------------------------------------- cases
def _layout(requests, context, new, ragged, pad, block, name=None):
    c = {"op": "layout", "requests": requests, "context": context, "new": new, "ragged": ragged, "pad": pad, "block": block}
    return {"name": name, **c} if name else c


def _adapters(rows, requests, slots, active, rank, hidden, q, kv, inter, none=0, name=None):
    c = {"op": "adapters", "rows": rows, "requests": requests, "slots": slots, "active": active, "rank": rank, "hidden": hidden, "q": q, "kv": kv,
         "inter": inter, "none": none}
    return {"name": name, **c} if name else c


def _draw(rows, vocab, kind, dtype="bfloat16", masked=False, name=None):
    c = {"op": "draw", "rows": rows, "vocab": vocab, "kind": kind, "dtype": dtype, "masked": masked}
    return {"name": name, **c} if name else c


def listed():
    return [
        # decode of a full server: one token a request, everything in one small launch
        _layout(256, 1280, 1, True, 256, 4, name="layout-decode-256"),
        # prefill: uneven portions of prompts fill a step of 8192 tokens
        _layout(37, 2048, 220, True, 0, 4, name="layout-prefill-37-ragged"),
        # long prompts of many requests at once, first page to last
        _layout(300, 8192, 700, True, 0, 2, name="layout-extend-300-long"),
        # one user with an adapter: latency
        _adapters(1, 1, 8, 1, 16, 4096, 4096, 1024, 12288, name="adapters-decode-1"),
        # a server at part load: 48 requests over 12 adapters, every fourth without one
        _adapters(48, 48, 16, 12, 32, 4096, 4096, 1024, 12288, none=4, name="adapters-decode-48"),
        # a full server, nearly every request with an adapter of its own choice
        _adapters(256, 256, 64, 64, 64, 4096, 4096, 1024, 12288, none=16, name="adapters-decode-256"),
        # one question arrives beside requests that decode: an odd number of rows, two adapters
        _adapters(331, 5, 8, 2, 16, 4096, 4096, 1024, 12288, name="adapters-prefill-331"),
        # prompts of eight requests over four adapters fill a step
        _adapters(8192, 8, 8, 4, 16, 4096, 4096, 1024, 12288, name="adapters-prefill-8192"),
        # one user who samples from the whole vocabulary
        _draw(1, 151936, "plain", name="draw-1-plain"),
        # users with settings of their own, grammars among them
        _draw(48, 151936, "mixed", masked=True, name="draw-48-mixed"),
        # a full server with the usual nucleus
        _draw(256, 151936, "top-p", name="draw-256-top-p"),
        # 32-bit logits of a small model with an odd vocabulary, settings mixed
        _draw(9, 50257, "mixed", "float32", name="draw-9-fp32"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["layout", "adapters", "adapters", "draw", "draw"])
    if op == "layout":
        if rng.random() < 0.4:
            n = log(2, 512)
            return _layout(n, log(1, 8192), 1, True, n + rng.randint(0, 64), rng.choice([1, 2, 4, 8, 16]))
        n = log(1, 300)
        return _layout(n, log(1, 8192), log(3, 200000 // n if n > 200 else 700), rng.random() < 0.8, 0, rng.choice([1, 2, 4, 8, 16]))
    if op == "adapters":
        slots = log(1, 64)
        rank = rng.choice([8, 16, 16, 24, 32, 64]) if slots > 8 else rng.choice([8, 16, 16, 32, 64, 128])
        hidden, kv = 64 * rng.randint(8, 64) + 8 * rng.randint(0, 1), 64 * rng.randint(1, 16)
        q, inter = kv * rng.choice([1, 2, 4]), 32 * rng.randint(16, 384)
        rows = log(1, 256) if slots > 16 or rng.random() < 0.5 else log(257, 4096)
        requests = rows if rows <= 256 else rng.randint(1, 12)
        return _adapters(rows, requests, slots, rng.randint(1, min(slots, requests)), rank, hidden, q, kv, inter, none=rng.choice([0, 0, 2, 5]))
    return _draw(log(1, 256), log(1000, 151936), rng.choice(["plain", "top-p", "mixed", "mixed"]), rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]),
                 rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------- inputs
def _generator(seed, where):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + where * 7919 + 17) % (1 << 40))


def _layout_lengths(case):
    """(tokens before the step, new tokens, pages held) of every request, on the host; a seed puts the requests in another order."""
    r = np.random.default_rng(3)
    n = case["requests"]
    start = np.full(n, case["context"]) if not case["ragged"] else r.integers(0, case["context"] + 1, n)
    count = np.ones(n, dtype=np.int64) if case["new"] == 1 else np.full(n, case["new"]) if not case["ragged"] else r.integers(0, 2 * case["new"] + 1, n)
    if case["new"] > 1 and count.sum() == 0:
        count[0] = 1
    # a request holds the pages of its context; one in eight was given its next pages a step ahead
    held = -(-start // PAGE) + (r.random(n) < 0.125) * r.integers(0, 3, n)
    return start, count, held


def _prepare_layout(case, seed):
    n = case["requests"]
    r = np.random.default_rng(seed * 104729 + 11)
    order = r.permutation(n)
    start, count, held = (v[order] for v in _layout_lengths(case))
    rows = n + 5
    width = int((-(-(start + count) // PAGE)).max().clip(int(held.max()))) + 4
    need = np.maximum(0, -(-(start + count) // PAGE) - held)
    ids = r.permutation(int(rows * width + need.sum()))
    table = np.full((rows, width), -1, dtype=np.int32)
    slots = r.permutation(rows)[:n]
    table[slots] = np.where(np.arange(width) < held[:, None], ids[:n * width].reshape(n, width), -1)
    pages = ids[n * width:n * width + int(need.sum())]
    block = case["block"]
    tokens, blocks = int(count.sum()), int((-(-count // block)).sum())
    t = {k: torch.from_numpy(np.ascontiguousarray(v.astype(np.int32))).cuda() for k, v in
         (("request", slots), ("start", start), ("count", count), ("held", held), ("pages", pages), ("table", table))}
    s = {**t, "tokens": tokens, "blocks": blocks, "pad": case["pad"], "block": block}
    if own:
        from cubic_serve_b200.ops import kernels as K
        s["layout"] = K.StepLayout(max(tokens, case["pad"]), n, max(blocks, case["pad"]), torch.device("cuda"))
    return s


def _projections(case):
    """(name, inputs, widths of the sections) of the projections of a layer."""
    h, q, kv, i = case["hidden"], case["q"], case["kv"], case["inter"]
    return (("qkv", h, (q, kv, kv)), ("o", q, (h,)), ("gate_up", h, (i, i)), ("down", i, (h,)))


def _row_adapters(case):
    """Adapter of every row (-1: none), on the host: request i takes one of the active adapters in turn."""
    req = np.sort(np.arange(case["rows"]) * case["requests"] // case["rows"])
    a = (req % case["active"]) * case["slots"] // case["active"]
    if case["none"]:
        a[req % case["none"] == case["none"] - 1] = -1
    if case["rows"] == case["requests"]:
        a = a[np.random.default_rng(5).permutation(case["rows"])]          # requests decode in the order in which they came
    return a.astype(np.int32)


def _prepare_adapters(case, seed):
    ids = torch.from_numpy(_row_adapters(case)).cuda()
    s = {"ids": ids, "slots": case["slots"]}
    for i, (name, k, widths) in enumerate(_projections(case)):
        g = _generator(seed, i)
        n, rank = sum(widths), case["rank"]

        def rnd(*shape, std):
            return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0, std, generator=g)

        a, b = rnd(case["slots"], len(widths) * rank, k, std=k ** -0.5), rnd(case["slots"], n, rank, std=0.05)
        scale = torch.rand(case["slots"], device="cuda", generator=g) + 0.5
        section = torch.repeat_interleave(torch.arange(len(widths)), torch.tensor(widths)).cuda()
        p = {"x": rnd(case["rows"], k, std=1.0), "y": rnd(case["rows"], n, std=1.0), "a": a, "b": b, "scale": scale, "section": section, "sections": len(widths)}
        if own:
            from cubic_serve_b200.ops import kernels as K
            p["bank"] = K.AdapterBank(a, b, scale, widths)
        s[name] = p
    if own:
        from cubic_serve_b200.ops import kernels as K
        s["rows"] = K.AdapterRows(case["rows"], case["slots"], 3 * case["rank"], torch.device("cuda"))
    return s


def _settings(case, seed):
    """temperature, top_k, top_p, min_p of every row, on the host."""
    n, kind = case["rows"], case["kind"]
    r = np.random.default_rng(seed * 31337 + 5)
    t = np.full(n, 1.0 if kind == "plain" else 0.7)
    k, p, m = np.zeros(n, dtype=np.int64), np.ones(n), np.zeros(n)
    if kind == "top-p":
        t, p = r.choice([0.6, 0.7, 1.0], n), r.choice([0.8, 0.9, 0.95], n)
    elif kind == "mixed":
        t = r.choice([0.0, 0.3, 0.7, 1.0, 1.5], n, p=[0.1, 0.2, 0.3, 0.3, 0.1])
        k, p, m = r.choice([0, 1, 20, 50, 200, 1000], n), r.choice([1.0, 0.5, 0.9, 0.99], n), r.choice([0.0, 0.0, 0.02, 0.1, 0.3], n)
    return t, k, p, m


def _prepare_draw(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    g = _generator(seed, 21)
    # a head's logits: a broad body, and a few tokens that stand out by as much as the context says
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 2.2 - 1.0
    hot = torch.arange(40, device="cuda") * (vocab // 40) + torch.randint(0, vocab // 40, (rows, 40), device="cuda", generator=g)
    x.scatter_(1, hot, 4.0 + 9.0 * torch.rand(rows, 40, device="cuda", generator=g))
    t, k, p, m = _settings(case, seed)
    s = {"logits": x.to(getattr(torch, case["dtype"])), "uniforms": torch.rand(rows, device="cuda", generator=g), "mask": None}
    s["temperature"], s["top_p"], s["min_p"] = (torch.from_numpy(v.astype(np.float32)).cuda() for v in (t, p, m))
    s["top_k"] = torch.from_numpy(k.astype(np.int32)).cuda()
    if case["masked"]:
        # every third row is under a grammar that allows about one token in fifty; bit i of the words is token i
        words = -(-vocab // 32)
        bits = torch.rand(rows, words * 32, device="cuda", generator=g) < 0.02
        bits[:, :4] = True
        bits[torch.arange(rows, device="cuda") % 3 != 0] = True
        s["mask"] = (bits.view(rows, words, 32).long() << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    s["ids"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    s["logprob"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    s["kept"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = {"layout": _prepare_layout, "adapters": _prepare_adapters, "draw": _prepare_draw}[case["op"]](case, seed)
    s["op"] = case["op"]
    return s


# ------------------------------------------------------------------------------------------------- the passes
LAYOUT = ("positions", "slots", "rb_req", "rb_qstart", "rb_qcount", "rb_ctx", "row0", "logit_rows")


def _plain_layout(s):
    start, count, held, pages, table, pad, block = s["start"].long(), s["count"].long(), s["held"].long(), s["pages"].long(), s["table"], s["pad"], s["block"]
    n, T, B, dev = start.numel(), s["tokens"], s["blocks"], start.device
    req = s["request"].long()
    need = ((start + count + PAGE - 1) // PAGE - held).clamp_min(0)
    upto = need.cumsum(0)
    if pages.numel():
        f = torch.arange(pages.numel(), device=dev)
        i = torch.searchsorted(upto, f, right=True)
        table[req[i], held[i] + f - (upto - need)[i]] = s["pages"]
    rows = count.cumsum(0)
    row0 = rows - count
    t = torch.arange(T, device=dev)
    i = torch.searchsorted(rows, t, right=True)
    pos = start[i] + t - row0[i]
    slots = table[req[i], pos // PAGE].long() * PAGE + pos % PAGE
    nb = (count + block - 1) // block
    b_upto = nb.cumsum(0)
    b = torch.arange(B, device=dev)
    j = torch.searchsorted(b_upto, b, right=True)
    first = (b - (b_upto - nb)[j]) * block
    out = {"positions": pos, "slots": slots, "rb_req": req[j], "rb_qstart": row0[j] + first, "rb_qcount": torch.minimum(count[j] - first, torch.full_like(first, block)),
           "rb_ctx": start[j] + first + 1, "row0": row0, "logit_rows": torch.where(count > 0, rows - 1, -1)}
    if pad > T:
        tail = torch.arange(T, pad, device=dev)
        zero = torch.zeros_like(tail)
        out["positions"], out["slots"] = torch.cat([pos, zero]), torch.cat([slots, zero - 1])
    if pad > B:
        tail = torch.arange(B, pad, device=dev)
        zero = torch.zeros_like(tail)
        out["rb_req"], out["rb_qstart"] = torch.cat([out["rb_req"], zero]), torch.cat([out["rb_qstart"], tail])
        out["rb_qcount"], out["rb_ctx"] = torch.cat([out["rb_qcount"], zero]), torch.cat([out["rb_ctx"], zero])
    out = {k: v if k == "logit_rows" else v.int() for k, v in out.items()}
    out["table"] = table
    return out


def _own_layout(s):
    from cubic_serve_b200.ops import kernels as K
    K.step_layout(s["request"], s["start"], s["count"], s["held"], s["pages"], s["table"], s["layout"], s["block"], tokens=s["tokens"], blocks=s["blocks"], pad=s["pad"])
    o, t, b, n = s["layout"], max(s["tokens"], s["pad"]), max(s["blocks"], s["pad"]), s["start"].numel()
    return {"positions": o.positions[:t], "slots": o.slots[:t], "rb_req": o.rb_req[:b], "rb_qstart": o.rb_qstart[:b], "rb_qcount": o.rb_qcount[:b], "rb_ctx": o.rb_ctx[:b],
            "row0": o.row0[:n], "logit_rows": o.logit_rows[:n], "table": s["table"]}


def _plain_adapter(p, ids):
    slots, r, k = p["a"].shape
    n, S = p["b"].shape[1], p["sections"]
    rank = r // S
    mine = ids[:, None] == torch.arange(slots, device=ids.device)                                       # [T, slots]
    h = (p["x"].float() @ p["a"].float().view(slots * r, k).t()).view(-1, slots, S, rank)
    h = torch.where(mine[:, :, None, None], h * p["scale"][:, None, None], 0.0).flatten(1)
    of = p["section"] == torch.arange(S, device=ids.device)[:, None]                                    # [S, n]: a section's columns see its own ranks
    b = torch.where(of[:, None, :], p["b"].float().transpose(1, 2)[:, None], 0.0).reshape(slots * r, n)
    return (p["y"].float() + h @ b).to(p["y"].dtype)


def _plain_adapters(s):
    return {"qkv": _plain_adapter(s["qkv"], s["ids"]), "o": _plain_adapter(s["o"], s["ids"]), "gate_up": _plain_adapter(s["gate_up"], s["ids"]),
            "down": _plain_adapter(s["down"], s["ids"])}


def _own_adapters(s):
    from cubic_serve_b200.ops import kernels as K
    rows = K.adapter_rows(s["ids"], s["rows"])

    def add(p):
        return K.adapter_add(p["x"], p["y"], p["bank"], rows, out=torch.empty_like(p["y"]))

    return {"qkv": add(s["qkv"]), "o": add(s["o"]), "gate_up": add(s["gate_up"]), "down": add(s["down"])}


def _plain_draw(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    dev = x.device
    ok = (x == x) & (x > -math.inf)
    if s["mask"] is not None:
        i = torch.arange(vocab, device=dev)
        ok &= ((s["mask"].long()[:, i // 32] >> (i % 32)) & 1).bool()
    x = torch.where(ok, x, -math.inf)
    v, order = torch.sort(x, dim=1, descending=True, stable=True)                                       # equal values: lowest id first
    t = s["temperature"].double()[:, None]
    top = v[:, :1]
    w = torch.where(v > -math.inf, torch.exp((v - top) / torch.where(t > 0, t, 1.0)), 0.0)
    at = torch.arange(vocab, device=dev)
    count = ok.sum(1, keepdim=True)
    k = s["top_k"].long()[:, None]
    n = torch.where(k > 0, torch.minimum(k, count), count)
    upto = w.cumsum(1)
    mass = upto.gather(1, (n - 1).clamp_min(0))
    p = s["top_p"].double()[:, None]
    n = torch.where(p < 1, torch.minimum(n, 1 + (upto < p * mass).sum(1, keepdim=True)), n)
    m = s["min_p"].double()[:, None]
    n = torch.where(m > 0, torch.minimum(n, ((w >= m) & (at < count)).sum(1, keepdim=True)), n)
    n = torch.where(t > 0, n, torch.minimum(count, torch.ones_like(n)))
    mass = upto.gather(1, (n - 1).clamp_min(0))
    pick = torch.minimum((upto <= s["uniforms"].double()[:, None] * mass).sum(1, keepdim=True), n - 1).clamp_min(0)
    logprob = torch.where(t > 0, torch.log(w.gather(1, pick) / mass), 0.0)
    return {"ids": order.gather(1, pick)[:, 0].int(), "logprob": logprob[:, 0].float(), "kept": n[:, 0].int()}


def _own_draw(s):
    from cubic_serve_b200.ops import kernels as K
    K.sample_vocabulary(s["logits"], s["ids"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], uniforms=s["uniforms"], mask=s["mask"], out_logprob=s["logprob"],
                        out_kept=s["kept"])
    return {"ids": s["ids"], "logprob": s["logprob"], "kept": s["kept"]}


def run(state):
    with torch.no_grad():
        if state["op"] == "layout":
            return _own_layout(state) if own else _plain_layout(state)
        if state["op"] == "adapters":
            return _own_adapters(state) if own else _plain_adapters(state)
        return _own_draw(state) if own else _plain_draw(state)


# ------------------------------------------------------------------------------------------------- work and truth
def work(case):
    if case["op"] == "layout":
        start, count, held = _layout_lengths(case)
        n, tokens, blocks = case["requests"], max(int(count.sum()), case["pad"]), max(int((-(-count // case["block"])).sum()), case["pad"])
        taken = int(np.maximum(0, -(-(start + count) // PAGE) - held).sum())
        seen = int((count > 0).sum() + count.sum() // PAGE)
        return {"bytes": n * (4 * 4 + 4 + 8) + taken * 8 + seen * 4 + tokens * 8 + blocks * 16, "flops": 0}
    if case["op"] == "adapters":
        ids = _row_adapters(case)
        used, rows = len(set(ids[ids >= 0].tolist())), int((ids >= 0).sum())
        nbytes = flops = 0
        for _, k, widths in _projections(case):
            n, r = sum(widths), len(widths) * case["rank"]
            nbytes += 2 * (used * (r * k + n * case["rank"]) + rows * k + 2 * case["rows"] * n)
            flops += 2 * rows * (r * k + n * case["rank"])
        return {"bytes": nbytes + 4 * case["rows"], "flops": flops}
    size = 2 if case["dtype"] == "bfloat16" else 4
    words = -(-case["vocab"] // 32) * 4 if case["masked"] else 0
    return {"bytes": case["rows"] * (case["vocab"] * size + words + 32), "flops": case["rows"] * case["vocab"] * 4}


def _exact_adapters(case, seed):
    s = prepare(case, seed)
    ids = _row_adapters(case)
    out = {}
    for name, _, widths in _projections(case):
        p, rank = s[name], case["rank"]
        y = p["y"].double()
        for slot in sorted(set(ids[ids >= 0].tolist())):
            rows = torch.from_numpy(np.flatnonzero(ids == slot)).cuda()
            x, col = p["x"][rows].double(), 0
            for i, width in enumerate(widths):
                a = p["a"][slot, i * rank:(i + 1) * rank].double()
                b = p["b"][slot, col:col + width].double()
                y[rows, col:col + width] += float(p["scale"][slot]) * ((x @ a.t()) @ b.t())
                col += width
        out[name] = y
    return out


def _exact_draw(case, seed):
    s = prepare(case, seed)
    x, u = s["logits"].double().cpu().numpy(), s["uniforms"].double().cpu().numpy()
    setting = [s[k].double().cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p")]
    mask = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint32)
    logprob = np.zeros(case["rows"])
    for r in range(case["rows"]):
        t, k, p, m = (float(v[r]) for v in setting)
        ids = np.arange(case["vocab"])
        if mask is not None:
            ids = ids[(mask[r][ids >> 5] >> (ids & 31)) & 1 == 1]
        ids = ids[np.argsort(-x[r][ids], kind="stable")]
        if t <= 0:
            continue
        if k > 0:
            ids = ids[:int(k)]
        w = np.exp((x[r][ids] - x[r][ids[0]]) / t)
        if p < 1:
            w = w[:1 + int(np.searchsorted(np.cumsum(w), p * math.fsum(w)))]
        if m > 0:
            w = w[w >= m]
        upto = np.cumsum(w)
        logprob[r] = math.log(w[min(int(np.searchsorted(upto, u[r] * upto[-1], side="right")), len(w) - 1)] / math.fsum(w))
    return {"ids": None, "logprob": torch.from_numpy(logprob), "kept": None}


def exact(case, seed):
    """Every number of the layout is a whole number: it has no other value in 64 bits."""
    if case["op"] == "layout":
        return None
    return _exact_adapters(case, seed) if case["op"] == "adapters" else _exact_draw(case, seed)
