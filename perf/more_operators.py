"""What a round of speculative decoding with a tree of drafts does, besides the shared layers, and what a request says about its tokens.

A round gives every request a tree of drafted tokens: node 0 is its last token, node j > 0 a draft that follows its parent.  The
target runs all nodes at once, their keys and values behind the request's context in the pages of the quantised cache.

* Attention of the nodes: every node sees the whole context and, of the tree, the nodes that its mask names (its ancestors and
  itself).  A pass is one layer.
* Logits as the requests want them: penalties for repeated tokens (with the drafts that lead to a node counted), biases of chosen
  tokens, the masks of grammars.
* The round's end: the path that the target agrees with, and its keys and values moved up behind the context, in all layers.

The plain forms are elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE, D, GROUP = 16, 128, 32


# ------------------------------------------------------------------------------------------------- cases
def _tree(requests, nodes, context, hq, hkv, k_bits, v_bits, ragged=False, name=None):
    c = {"op": "tree", "requests": requests, "nodes": nodes, "context": context, "hq": hq, "hkv": hkv, "k_bits": k_bits, "v_bits": v_bits, "ragged": ragged}
    return {"name": name, **c} if name else c


def _wishes(requests, nodes, vocab, history, bias=0, masked=0, dtype="bfloat16", name=None):
    c = {"op": "wishes", "requests": requests, "nodes": nodes, "vocab": vocab, "history": history, "bias": bias, "masked": masked, "dtype": dtype}
    return {"name": name, **c} if name else c


def _keep(requests, nodes, context, layers, hkv, k_bits, v_bits, name=None):
    c = {"op": "keep", "requests": requests, "nodes": nodes, "context": context, "layers": layers, "hkv": hkv, "k_bits": k_bits, "v_bits": v_bits}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user, a few drafts: latency
        _tree(1, 8, 700, 32, 8, 8, 8, name="tree-1x8"),
        # a handful of users, trees of uneven sizes behind uneven contexts
        _tree(7, 26, 2100, 32, 8, 8, 8, ragged=True, name="tree-7x26-ragged"),
        # a server at part load with narrow trees
        _tree(64, 16, 4096, 32, 8, 8, 8, name="tree-64x16"),
        # wide trees over few key / value heads, six bits
        _tree(32, 64, 1500, 64, 4, 6, 6, ragged=True, name="tree-32x64-six-bits"),
        # two long documents, keys in four bits
        _tree(2, 64, 32000, 32, 4, 4, 8, name="tree-2x64-long"),
        # one user with penalties
        _wishes(1, 1, 151936, 900, name="wishes-1"),
        # a full server: penalties everywhere, some biases, some grammars
        _wishes(256, 1, 151936, 1280, bias=60, masked=8, name="wishes-256"),
        # the rows of trees, each behind drafts of its own
        _wishes(24, 26, 151936, 1500, bias=20, name="wishes-24x26-trees"),
        # 32-bit logits of a small model with an odd vocabulary, long histories
        _wishes(9, 1, 50257, 20000, bias=300, masked=3, dtype="float32", name="wishes-9-fp32"),
        # one user's round ends
        _keep(1, 8, 700, 36, 8, 8, 8, name="keep-1x8"),
        # a server's, eight bits
        _keep(64, 26, 1500, 12, 8, 8, 8, name="keep-64x26"),
        # a full server's, keys in four bits
        _keep(256, 16, 900, 12, 4, 4, 8, name="keep-256x16-four-bits"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    bits = rng.choice([(8, 8), (8, 8), (4, 8), (6, 6), (4, 4), (8, 4)])
    op = rng.choice(["tree", "tree", "wishes", "wishes", "keep"])
    if op == "tree":
        hq, hkv = rng.choice([(32, 8), (32, 8), (32, 4), (64, 4), (28, 4), (16, 16), (8, 1)])
        n, nodes = log(1, 64), log(1, 100)
        return _tree(n, nodes, log(16, max(17, min(30000, 2000000 // (n * hkv), 32000000 // (n * nodes * hq)))), hq, hkv, *bits, ragged=rng.random() < 0.6)
    if op == "wishes":
        n = log(1, 256)
        vocab = log(1000, 151936)
        nodes = 1 if rng.random() < 0.5 else log(2, max(2, min(64, 600 // n)))
        return _wishes(n, nodes, vocab, log(1, 30000 if n < 16 else 3000), bias=rng.choice([0, 0, 20, 300]), masked=rng.choice([0, 0, 2, 5]),
                       dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    n = log(1, 256)
    return _keep(n, log(2, 64), log(1, 3000), rng.randint(1, 6 if n > 64 else 24), rng.choice([2, 4, 8]), *bits)


# ------------------------------------------------------------------------------------------------- inputs
def _generator(seed, where):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + where * 7919 + 29) % (1 << 40))


def _i32(v):
    return torch.from_numpy(np.ascontiguousarray(v).astype(np.int32)).cuda()


def _parents(n, r):
    """A tree of ``n`` nodes level by level: the parent of every node, -1 for node 0.  Near the root it is wider than it is deep."""
    p = np.zeros(n, dtype=np.int64)
    p[0] = -1
    wide = min(n, 6)
    for j in range(wide, n):
        p[j] = max(p[j - 1], int(r.integers(0, max(1, int(0.7 * j)))))
    return p


def _ancestors(parents):
    """[n, n] truth values: node i sees node j."""
    n = len(parents)
    m = np.eye(n, dtype=bool)
    for j in range(1, n):
        m[j] |= m[parents[j]]
    return m


def _words(m, words):
    """Rows of truth values as 32-bit words, bit i of word w = column 32 w + i."""
    full = np.zeros((m.shape[0], words * 32), dtype=np.uint64)
    full[:, :m.shape[1]] = m
    return (full.reshape(m.shape[0], words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def _sizes(case):
    """(nodes, context) of every request, on the host; a seed puts them in another order."""
    r = np.random.default_rng(17)
    n = case["requests"]
    if not case.get("ragged"):
        return np.full(n, case["nodes"]), np.full(n, case["context"])
    nodes, context = r.integers(max(1, case["nodes"] // 3), case["nodes"] + 1, n), r.integers(case["context"] // 3, case["context"] + 1, n)
    nodes[0], context[0] = case["nodes"], case["context"]
    return nodes, context


def _blob(hkv, k_bits, v_bits):
    return PAGE * D * (k_bits + v_bits) // 8 + 2 * PAGE * (D // GROUP) * 4


def _pack(codes, bits, keys):
    """Codes [pages, heads, 16 tokens, 128 channels], counted from zero, as the bytes of the cache (K or V)."""
    n, h = codes.shape[:2]
    c = codes.to(torch.uint8)
    swizzle = torch.arange(32, device=c.device)[None] ^ ((torch.arange(8, device=c.device) & 3) << 2)[:, None]            # place -> chunk
    if keys:
        if bits == 8:
            return c.view(n, h, 16, 8, 16).transpose(2, 3).reshape(n, h, -1)
        b = c.view(n, h, 16, 4, 2, 16).permute(0, 1, 3, 2, 4, 5)                                                          # block, token, half, 16
        low = ((b[..., 0, :] & 15) | ((b[..., 1, :] & 15) << 4)).reshape(n, h, -1)
        if bits == 4:
            return low
        f = b >> 4                                                                                                       # two bits
        w = (f[:, :, :, :8, 0] << 4) | (f[:, :, :, :8, 1] << 6) | f[:, :, :, 8:, 0] | (f[:, :, :, 8:, 1] << 2)
        return torch.cat([low, w.reshape(n, h, -1)], -1)
    v = c.view(n, h, 8, 2, 32, 4)                                                                                        # pair, token, chunk, channel
    v = torch.gather(v, 4, swizzle[None, None, :, None, :, None].expand(n, h, 8, 2, 32, 4))
    if bits == 8:
        return v.permute(0, 1, 2, 4, 5, 3).reshape(n, h, -1)
    low = ((v[:, :, :, 0] & 15) | ((v[:, :, :, 1] & 15) << 4)).reshape(n, h, -1)
    if bits == 4:
        return low
    f = v >> 4
    w = (f[:, :, :4, 0] << 4) | (f[:, :, :4, 1] << 6) | f[:, :, 4:, 0] | (f[:, :, 4:, 1] << 2)
    return torch.cat([low, w.reshape(n, h, -1)], -1)


def _cache(pages, hkv, k_bits, v_bits, g):
    """Pages of a cache as a server fills them: keys with a few channels that stand out, values without."""
    out = torch.empty(pages, hkv, _blob(hkv, k_bits, v_bits), dtype=torch.uint8, device="cuda")
    spread = 1 + 4 * (torch.arange(D, device="cuda") % 37 == 5)
    for a in range(0, pages, 4096):
        n, at = min(4096, pages - a), 0
        for bits, keys in ((k_bits, True), (v_bits, False)):
            x = torch.randn(n, hkv, 16, D, device="cuda", generator=g)
            if keys:
                x = x * spread
            x = x.view(n, hkv, 16, 4, GROUP)
            most = 2 ** (bits - 1) - 1
            scale = x.abs().amax(-1, keepdim=True) / most
            codes = (torch.round(x / scale).clamp(-most, most) + 2 ** (bits - 1)).view(n, hkv, 16, D)
            b = PAGE * D * bits // 8
            out[a:a + n, :, at:at + b] = _pack(codes, bits, keys)
            out[a:a + n, :, at + b:at + b + 256] = scale.reshape(n, hkv, 64).contiguous().view(torch.uint8).view(n, hkv, 256)
            at += b + 256
    return out


def _prepare_tree(case, seed):
    r = np.random.default_rng(seed * 104729 + 3)
    g = _generator(seed, 1)
    order = r.permutation(case["requests"])
    nodes, context = (v[order] for v in _sizes(case))
    n, total = case["requests"], int(nodes.sum())
    held = -(-(context + nodes) // PAGE)
    width = int(held.max()) + 2
    ids = r.permutation(int(held.sum()) + 3)
    table = np.full((n + 2, width), -1, dtype=np.int64)
    slots = r.permutation(n + 2)[:n]
    at = np.concatenate([[0], held.cumsum()])
    for i in range(n):
        table[slots[i], :held[i]] = ids[at[i]:at[i + 1]]
    words = -(-case["nodes"] // 32)
    masks = np.concatenate([_words(_ancestors(_parents(int(c), r)), words) for c in nodes])
    s = {k: case[k] for k in ("hq", "hkv", "k_bits", "v_bits")}
    s["cache"] = _cache(int(held.sum()) + 3, case["hkv"], case["k_bits"], case["v_bits"], g)
    s["q"] = torch.empty(total, case["hq"] * D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    s["out"] = torch.empty_like(s["q"])
    s["table"], s["request"], s["count"], s["start"], s["masks"] = _i32(table), _i32(slots), _i32(nodes), _i32(context), _i32(masks)
    s["row0"] = _i32(np.concatenate([[0], nodes.cumsum()[:-1]]))
    s["host"] = [(int(slots[i]), int(nodes[i]), int(context[i])) for i in range(n)]           # the scheduler's own copy
    return s


def _prepare_wishes(case, seed):
    r = np.random.default_rng(seed * 31337 + 7)
    g = _generator(seed, 2)
    n, nodes, vocab, rows = case["requests"], case["nodes"], case["vocab"], case["requests"] * case["nodes"]
    x = torch.randn(rows, vocab, device="cuda", generator=g) * 2.2 - 1.0
    s = {"logits": x.to(getattr(torch, case["dtype"])), "request": _i32(np.repeat(np.arange(n), nodes)), "nodes": nodes}
    s["out"] = torch.empty_like(s["logits"])
    # a history says some tokens again and again; the prompt is its first half or so
    length = r.integers(max(1, case["history"] // 2), case["history"] + 1, n)
    common = (vocab * r.random((n, case["history"])) ** 4).astype(np.int64)
    s["history"], s["length"], s["prompt"] = _i32(common.clip(0, vocab - 1)), _i32(length), _i32((length * r.uniform(0.2, 1.0, n)).astype(np.int64))
    for k, choices in (("repetition", [1.0, 1.1, 1.3]), ("frequency", [0.0, 0.2, 0.7]), ("presence", [0.0, 0.3, 1.0])):
        v = r.choice(choices, n)
        v[:1] = choices[1]
        s[k] = torch.from_numpy(v.astype(np.float32)).cuda()
    s["bias"] = s["mask"] = s["drafts"] = None
    if case["bias"]:
        # every third request has biases
        count = np.where(np.arange(n) % 3 == 0, np.minimum(case["bias"], vocab // 2), 0)
        at = np.concatenate([[0], count.cumsum()])
        ids = np.concatenate([r.choice(vocab, int(c), replace=False) for c in count])
        s["bias"] = (_i32(at), _i32(ids), torch.from_numpy(r.uniform(-8, 8, len(ids)).astype(np.float32)).cuda())
    if case["masked"]:
        # some requests are under a grammar that allows about one token in fifty; bit i of the words is token i
        words = -(-vocab // 32)
        bits = torch.rand(rows, words * 32, device="cuda", generator=g) < 0.02
        bits[s["request"].long() % case["masked"] != 0] = True
        s["mask"] = (bits.view(rows, words, 32).long() << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    if nodes > 1:
        words = -(-nodes // 32)
        masks = np.concatenate([_words(_ancestors(_parents(nodes, r)), words) for _ in range(n)])
        tokens = (vocab * r.random(rows) ** 4).astype(np.int64).clip(0, vocab - 1)
        s["drafts"] = (_i32(tokens), _i32(masks), _i32(np.arange(n) * nodes))
    return s


def _prepare_keep(case, seed):
    r = np.random.default_rng(seed * 7907 + 13)
    g = _generator(seed, 3)
    n, nodes, context = case["requests"], case["nodes"], case["context"]
    held = -(-(context + nodes) // PAGE)
    first = context // PAGE                                                 # the cache of this process holds the last pages of every request
    own_pages = held - first
    ids = r.permutation(n * own_pages + 1)[:n * own_pages].reshape(n, own_pages)
    table = np.full((n, held + 1), -1, dtype=np.int64)
    table[:, :first] = 0
    table[:, first:held] = ids
    parents = np.stack([_parents(nodes, r) for _ in range(n)])
    tokens, target = r.integers(0, 151936, (n, nodes)), r.integers(0, 151936, (n, nodes))
    for i in range(n):
        # the target agrees with up to four drafts in a row: the first branch, or one whose nodes lie behind the places that they move to
        cur, first = 0, r.random() < 0.25
        for depth in range(4):
            c = np.flatnonzero(parents[i] == cur)
            c = c[c == depth + 1] if first else c[c >= min(5, nodes - 1)]
            if not len(c) or r.random() < 0.15:
                break
            nxt = int(r.choice(c))
            target[i, cur], cur = tokens[i, nxt], nxt
    s = {k: case[k] for k in ("hkv", "k_bits", "v_bits", "nodes")}
    s["cache"] = torch.stack([_cache(n * own_pages + 1, case["hkv"], case["k_bits"], case["v_bits"], g) for _ in range(case["layers"])])
    s["table"], s["request"], s["start"], s["count"], s["row0"] = _i32(table), _i32(np.arange(n)), _i32(np.full(n, context)), _i32(np.full(n, nodes)), _i32(np.arange(n) * nodes)
    s["parents"], s["tokens"], s["target"] = _i32(parents.reshape(-1)), _i32(tokens.reshape(-1)), _i32(target.reshape(-1))
    s["accepted"] = torch.empty(n, dtype=torch.int32, device="cuda")
    s["path"], s["emitted"] = (torch.empty(n, nodes, dtype=torch.int32, device="cuda") for _ in range(2))
    if own:
        from cubic_serve_b200.ops import kernels as K
        s["caches"] = K.LayerCaches(list(s["cache"]), case["hkv"], D, case["k_bits"], case["v_bits"])
    return s


def prepare(case, seed):
    s = {"tree": _prepare_tree, "wishes": _prepare_wishes, "keep": _prepare_keep}[case["op"]](case, seed)
    s["op"] = case["op"]
    return s


# ------------------------------------------------------------------------------------------------- the passes
def _unpack(raw, bits, keys):
    """The reverse of the cache's order: bytes [pages, heads, ...] -> signed codes [pages, heads, 16, 128], fp32."""
    n, h = raw.shape[:2]
    low = raw[..., :PAGE * D * min(bits, 8 if bits == 8 else 4) // 8]
    high = raw[..., PAGE * D // 2:PAGE * D * 6 // 8] if bits == 6 else None
    if keys:
        if bits == 8:
            c = low.reshape(n, h, 8, 16, 16).transpose(2, 3).reshape(n, h, 16, D)
        else:
            b = low.reshape(n, h, 4, 16, 16)
            two = torch.stack([b & 15, b >> 4], 4)                                       # block, token, half, 16
            if high is not None:
                w = high.reshape(n, h, 4, 8, 16)
                hi = torch.stack([torch.cat([w >> 4, w], 3), torch.cat([w >> 6, w >> 2], 3)], 4) & 3
                two = two | (hi << 4)
            c = two.permute(0, 1, 3, 2, 4, 5).reshape(n, h, 16, D)
    else:
        place = torch.arange(32, device=raw.device)[None] ^ ((torch.arange(8, device=raw.device) & 3) << 2)[:, None]
        if bits == 8:
            v = low.reshape(n, h, 8, 32, 4, 2).permute(0, 1, 2, 5, 3, 4)                 # pair, token, place, channel
        else:
            b = low.reshape(n, h, 8, 32, 4)
            v = torch.stack([b & 15, b >> 4], 3)
            if high is not None:
                w = high.reshape(n, h, 4, 32, 4)
                hi = torch.stack([torch.cat([w >> 4, w], 2), torch.cat([w >> 6, w >> 2], 2)], 3) & 3
                v = v | (hi << 4)
        c = torch.gather(v, 4, place[None, None, :, None, :, None].expand(n, h, 8, 2, 32, 4)).reshape(n, h, 16, D)
    return c.float() - 2 ** (bits - 1)


def _values(pages, k_bits, v_bits):
    """Keys and values [tokens, heads, 128] of pages of the cache, in 32 bits."""
    kb, vb = PAGE * D * k_bits // 8, PAGE * D * v_bits // 8
    n, h = pages.shape[:2]
    out = []
    for at, bits, keys, b in ((0, k_bits, True, kb), (kb + 256, v_bits, False, vb)):
        scale = pages[..., at + b:at + b + 256].contiguous().view(torch.float32).view(n, h, 16, 4, 1)
        x = _unpack(pages[..., at:at + b], bits, keys).view(n, h, 16, 4, GROUP) * scale
        out.append(x.view(n, h, 16, D).transpose(1, 2).reshape(n * 16, h, D))
    return out


def _plain_tree(s):
    hq, hkv = s["hq"], s["hkv"]
    bit, row = torch.arange(32, device="cuda"), 0
    for slot, c, context in s["host"]:
        total = context + c
        k, v = _values(s["cache"][s["table"][slot, :-(-total // PAGE)].long()], s["k_bits"], s["v_bits"])
        k, v = k[:total].transpose(0, 1), v[:total].transpose(0, 1)                      # [hkv, total, 128]
        q = s["q"][row:row + c].float().view(c, hkv, hq // hkv, D).transpose(0, 1).reshape(hkv, -1, D)
        x = (q @ k.transpose(1, 2)).view(hkv, c, hq // hkv, total) * (1 / math.sqrt(D))
        sees = ((s["masks"][row:row + c, :, None] >> bit) & 1).bool().view(c, -1)[:, :c]
        x[..., context:].masked_fill_(~sees[:, None], -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top > -math.inf, top, 0.0))
        mass = p.sum(-1, keepdim=True)
        p = torch.where(mass > 0, p / mass, 0.0).view(hkv, -1, total)
        s["out"][row:row + c] = (p @ v).view(hkv, c, hq // hkv, D).transpose(0, 1).reshape(c, hq * D)
        row += c
    return s["out"]


def _own_tree(s):
    from cubic_serve_b200.ops import kernels as K
    return K.tree_attention(s["q"], s["out"], s["cache"], s["table"], s["request"], s["row0"], s["count"], s["start"], s["masks"], s["hq"], s["hkv"], D, s["k_bits"], s["v_bits"])


def _plain_wishes(s):
    logits, req = s["logits"], s["request"].long()
    rows, vocab = logits.shape
    dev = logits.device
    at = torch.arange(s["history"].shape[1], device=dev)
    n = s["length"].numel()
    there = at < s["length"].long()[:, None]
    new = there & (at >= s["prompt"].long()[:, None])
    ids = s["history"].long()
    count = torch.zeros(n, vocab, device=dev).scatter_add_(1, ids, new.float())[req]
    seen = torch.zeros(n, vocab, device=dev).scatter_add_(1, ids, there.float())[req] > 0
    if s["drafts"] is not None:
        tokens, masks, row0 = s["drafts"]
        first = row0.long()[req]
        sees = ((masks[:, :, None] >> torch.arange(32, device=dev)) & 1).bool().view(rows, -1)
        j = torch.arange(s["nodes"], device=dev)
        extra = sees[:, 1:s["nodes"]].float()
        count.scatter_add_(1, tokens.long()[first[:, None] + j[1:]], extra)
        seen |= count > 0
    x = logits.float()
    rep = s["repetition"][req][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][req][:, None] * count
    x = x - torch.where(count > 0, s["presence"][req][:, None], 0.0)
    if s["bias"] is not None:
        start, ids, values = s["bias"]
        of = torch.searchsorted(start.long()[1:], torch.arange(ids.numel(), device=dev), right=True)
        add = torch.zeros(n, vocab, device=dev)
        add[of, ids.long()] = values
        x = x + add[req]
    if s["mask"] is not None:
        i = torch.arange(vocab, device=dev)
        x = torch.where(((s["mask"][:, i // 32] >> (i % 32).int()) & 1).bool(), x, -math.inf)
    s["out"].copy_(x)
    return s["out"]


def _own_wishes(s):
    from cubic_serve_b200.ops import kernels as K
    return K.adjust_logits(s["logits"], s["request"], s["history"], s["length"], s["prompt"], s["repetition"], s["frequency"], s["presence"], bias=s["bias"], mask=s["mask"],
                           drafts=s["drafts"], out=s["out"])


def _plain_keep(s):
    n, nodes, dev = s["start"].numel(), s["nodes"], s["start"].device
    parents, tokens, target = (s[k].view(n, nodes).long() for k in ("parents", "tokens", "target"))
    i, j = torch.arange(n, device=dev), torch.arange(nodes, device=dev)
    path, emitted = torch.full((n, nodes), -1, device=dev), torch.full((n, nodes), -1, device=dev)
    cur, going, accepted = torch.zeros_like(i), torch.ones_like(i).bool(), torch.zeros_like(i)
    for d in range(nodes):
        path[:, d] = torch.where(going, cur, -1)
        emitted[:, d] = torch.where(going, target[i, cur], -1)
        fits = (parents == cur[:, None]) & (tokens == target[i, cur][:, None]) & (j > 0) & going[:, None]
        going = fits.any(1)
        cur = torch.where(going, torch.where(fits, j, nodes).amin(1).clamp_max(nodes - 1), cur)
        accepted += going
    # a token's bytes: whole ones where it has them alone, else the bits of its half
    k, d = torch.meshgrid(i, j[1:], indexing="ij")
    moves = (path[:, 1:] > 0) & (path[:, 1:] != d)
    req, to, of = k[moves], d[moves], path[:, 1:][moves]
    src, dst = s["start"].long()[req] + of, s["start"].long()[req] + to
    table = s["table"].long()
    _move_lines(s["cache"], table[s["request"].long()[req], src // PAGE], src % PAGE, table[s["request"].long()[req], dst // PAGE], dst % PAGE, s["k_bits"], s["v_bits"])
    s["accepted"].copy_(accepted)
    s["path"].copy_(path)
    s["emitted"].copy_(emitted)
    return {"accepted": s["accepted"], "path": s["path"], "emitted": s["emitted"], "cache": s["cache"]}


def _move_lines(cache, src_page, src, dst_page, dst, k_bits, v_bits):
    """Tokens one place after the other: a path's places rise, so each is read before anything is put there."""
    kb, vb = PAGE * D * k_bits // 8, PAGE * D * v_bits // 8
    if not src.numel():
        return
    m = torch.arange(src.numel(), device=src.device)
    a, b = cache[:, src_page], cache[:, dst_page]                                        # [layers, moves, heads, bytes]
    pages, which = torch.unique(dst_page, return_inverse=True)                           # moves into one page meet there
    to = cache[:, pages]
    layers, _, hkv, _ = a.shape
    for at, bits, keys, size in ((0, k_bits, True, kb), (kb + 256, v_bits, False, vb)):
        x = _unpack(a[..., at:at + size].flatten(0, 1), bits, keys).view(layers, -1, hkv, 16, D)[:, m, :, src]
        y = _unpack(to[..., at:at + size].flatten(0, 1), bits, keys).view(layers, -1, hkv, 16, D)
        y[:, which, :, dst] = x
        to[..., at:at + size] = _pack((y + 2 ** (bits - 1)).flatten(0, 1), bits, keys).view(layers, -1, hkv, size)
        x = a[..., at + size:at + size + 256].reshape(layers, -1, hkv, 16, 16)[:, m, :, src]
        y = to[..., at + size:at + size + 256].reshape(layers, -1, hkv, 16, 16)
        y[:, which, :, dst] = x
        to[..., at + size:at + size + 256] = y.reshape(layers, -1, hkv, 256)
    cache[:, pages] = to


def _own_keep(s):
    from cubic_serve_b200.ops import kernels as K
    K.verify_tree(s["target"], s["tokens"], s["parents"], s["row0"], s["count"], s["accepted"], s["path"], s["emitted"])
    K.keep_tokens(s["caches"], s["table"], s["request"], s["start"], s["accepted"], s["path"])
    return {"accepted": s["accepted"], "path": s["path"], "emitted": s["emitted"], "cache": s["cache"]}


def run(state):
    with torch.no_grad():
        if state["op"] == "tree":
            return _own_tree(state) if own else _plain_tree(state)
        if state["op"] == "wishes":
            return _own_wishes(state) if own else _plain_wishes(state)
        return _own_keep(state) if own else _plain_keep(state)


# ------------------------------------------------------------------------------------------------- work and truth
def work(case):
    if case["op"] == "tree":
        nodes, context = _sizes(case)
        hq, hkv = case["hq"], case["hkv"]
        tokens, rows = int((nodes + context).sum()), int(nodes.sum())
        line = D * (case["k_bits"] + case["v_bits"]) // 8 + 2 * (D // GROUP) * 4
        pages = int((-(-(nodes + context) // PAGE)).sum())
        return {"bytes": tokens * hkv * line + 4 * rows * hq * D + rows * -(-case["nodes"] // 32) * 4 + 4 * pages,
                "flops": 4 * D * hq * int((nodes * context + np.minimum(nodes * 5, nodes * nodes)).sum())}
    if case["op"] == "wishes":
        size = 2 if case["dtype"] == "bfloat16" else 4
        rows = case["requests"] * case["nodes"]
        words = -(-case["vocab"] // 32) * 4 if case["masked"] else 0
        return {"bytes": rows * (2 * case["vocab"] * size + words) + case["requests"] * (3 * case["history"] + 24), "flops": rows * case["vocab"]}
    # about two and a half drafts are accepted, three quarters of them move; a line is read and written
    line = D * (case["k_bits"] + case["v_bits"]) // 8 + 2 * (D // GROUP) * 4
    return {"bytes": case["requests"] * (case["nodes"] * 12 + int(1.9 * case["layers"] * case["hkv"] * 2 * line)), "flops": 0}


def _codes64(raw, bits, keys):
    """Signed codes [16, 128] of a page and head, element by element through the places that the cache's order gives."""
    t, c = torch.meshgrid(torch.arange(16, device=raw.device), torch.arange(D, device=raw.device), indexing="ij")
    if keys:
        at = c // 16 * 256 + t * 16 + c % 16 if bits == 8 else c // 32 * 256 + t * 16 + c % 16
        shift, high = c % 32 // 16 * 4, 1024 + c // 32 * 128 + t % 8 * 16 + c % 16
        high_shift = torch.where(t < 8, 4, 0) + c % 32 // 16 * 2
    else:
        place = (c // 4) ^ ((t // 2 % 4) * 4)
        at = t // 2 * 256 + place * 8 + c % 4 * 2 + t % 2 if bits == 8 else t // 2 * 128 + place * 4 + c % 4
        shift, high = t % 2 * 4, 1024 + t // 2 % 4 * 128 + place * 4 + c % 4
        high_shift = torch.where(t < 8, 4, 0) + t % 2 * 2
    x = raw[..., at.reshape(-1)].int()
    if bits < 8:
        x = (x >> shift.reshape(-1).int()) & 15
    if bits == 6:
        x = x | ((raw[..., high.reshape(-1)].int() >> high_shift.reshape(-1).int()) & 3) << 4
    return (x - 2 ** (bits - 1)).view(*raw.shape[:-1], 16, D)


def _exact_tree(case, seed):
    s = prepare(case, seed)
    hq, hkv, kb, vb = case["hq"], case["hkv"], case["k_bits"], case["v_bits"]
    out, row = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    masks = s["masks"].cpu().numpy().view(np.uint32)
    for slot, c, context in s["host"]:
        total = context + c
        blobs = s["cache"][s["table"][slot, :-(-total // PAGE)].long()]
        sees = torch.ones(c, total, dtype=torch.bool)
        for i in range(c):
            for j in range(c):
                sees[i, context + j] = bool(masks[row + i, j // 32] >> np.uint32(j % 32) & 1)
        sees = sees.cuda()
        for h in range(hkv):
            b, kv, at = blobs[:, h], [], 0
            for bits, keys in ((kb, True), (vb, False)):
                size = 256 * bits
                scale = b[:, at + size:at + size + 256].contiguous().view(torch.float32).view(-1, 16, 4).double().repeat_interleave(GROUP, -1)
                kv.append((_codes64(b[:, at:at + size], bits, keys).double() * scale).view(-1, D)[:total])
                at += size + 256
            for g in range(hq // hkv):
                col = (h * (hq // hkv) + g) * D
                x = s["q"][row:row + c, col:col + D].double() @ kv[0].t() / math.sqrt(D)
                p = torch.softmax(x.masked_fill(~sees, -math.inf), -1)
                out[row:row + c, col:col + D] = torch.nan_to_num(p) @ kv[1]
        row += c
    return out


def _exact_wishes(case, seed):
    s = prepare(case, seed)
    x = s["logits"].double().cpu().numpy()
    h = {k: s[k].cpu().numpy() for k in ("request", "history", "length", "prompt")}
    rep, freq, pres = (s[k].double().cpu().numpy() for k in ("repetition", "frequency", "presence"))
    bias = None if s["bias"] is None else [t.cpu().numpy() for t in s["bias"]]
    mask = None if s["mask"] is None else s["mask"].cpu().numpy().view(np.uint32)
    drafts = None if s["drafts"] is None else [t.cpu().numpy() for t in s["drafts"]]
    for r in range(x.shape[0]):
        q = int(h["request"][r])
        said = h["history"][q, :h["length"][q]]
        new = said[h["prompt"][q]:]
        if drafts is not None:
            first = int(drafts[2][q])
            more = [drafts[0][first + j] for j in range(1, case["nodes"]) if drafts[1].view(np.uint32)[r, j // 32] >> np.uint32(j % 32) & 1]
            said, new = np.concatenate([said, more]), np.concatenate([new, more])
        ids = np.unique(said.astype(np.int64))
        x[r, ids] = np.where(x[r, ids] > 0, x[r, ids] / rep[q], x[r, ids] * rep[q])
        ids, times = np.unique(new.astype(np.int64), return_counts=True)
        x[r, ids] -= freq[q] * times + pres[q]
        if bias is not None:
            a, b = bias[0][q], bias[0][q + 1]
            x[r, bias[1][a:b]] += bias[2][a:b].astype(np.float64)
        if mask is not None:
            i = np.arange(case["vocab"])
            x[r, (mask[r][i >> 5] >> (i & 31).astype(np.uint32)) & 1 == 0] = -math.inf
    return torch.from_numpy(x)


def exact(case, seed):
    """What a round keeps is whole numbers and bytes: they have no other value in 64 bits."""
    if case["op"] == "keep":
        return None
    return _exact_tree(case, seed) if case["op"] == "tree" else _exact_wishes(case, seed)
