"""Operators of a decoder's serving step: rotary positions with the append to a paged cache, attention
whose scores are capped, biased or masked by rules, attention of drafted tokens over the cache, and the
choice of a token from the logits.

`run` is one call of one operator: the framework's (`own`), or its plain form in elementary torch
operations, 32 bits throughout and 64 where 32 lose what matters (angles of far positions, sums next to
a border of the sampling).  `exact` computes the same from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def _rotary(name, tokens, heads, kv_heads, head, rot, layout, dtype, page, longest, scaling):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head": head, "rot": rot,
            "layout": layout, "dtype": dtype, "page": page, "longest": longest, "scaling": scaling}


def _rules(name, batch, heads, kv_heads, length, head, dtype, causal, cap, bias, documents, prefix):
    return {"name": name, "op": "rules", "batch": batch, "heads": heads, "kv_heads": kv_heads, "length": length, "head": head,
            "dtype": dtype, "causal": causal, "cap": cap, "bias": bias, "documents": documents, "prefix": prefix}


def _tree(name, requests, longest, drafts, heads, kv_heads, head, dtype, page, cap, bias):
    return {"name": name, "op": "tree", "requests": requests, "longest": longest, "drafts": drafts, "heads": heads,
            "kv_heads": kv_heads, "head": head, "dtype": dtype, "page": page, "cap": cap, "bias": bias}


def _sample(name, rows, vocab, dtype, top_k, top_p, min_p, masked):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "masked": masked}


def listed():
    return [
        # one decoding step of eight requests to the benchmark's decoder: a quarter of each head turns, latency counts
        _rotary("rotary_step_t8_f32", 8, 16, 16, 64, 16, "halves", "f32", 16, 2048, "plain"),
        # a long prompt at far positions, grouped heads, keys and values into the cache
        _rotary("rotary_prompt_t8191_bf16", 8191, 32, 8, 128, 128, "interleaved", "bf16", 64, 131072, "ramp"),
        # a short prompt of odd length to the benchmark's decoder, scores biased by distance
        _rules("rules_b1_s77_f32", 1, 16, 16, 77, 64, "f32", True, 0.0, True, 0, False),
        # the benchmark's four prompts of 512 tokens, each with a part that sees both ways
        _rules("rules_b4_s512_f32", 4, 16, 16, 512, 64, "f32", True, 0.0, False, 0, True),
        # middle-sized prompts in half precision: distance bias and prefix at once
        _rules("rules_b4_s2048_f16", 4, 16, 16, 2048, 64, "f16", True, 0.0, True, 0, True),
        # documents packed into one long row, capped scores, grouped heads
        _rules("rules_packed_s8191_bf16", 1, 32, 8, 8191, 128, "bf16", True, 50.0, False, 5, False),
        # one token of one conversation: the smallest serving step
        _tree("tree_r1_n1_bf16", 1, 1000, 1, 32, 8, 128, "bf16", 16, 0.0, False),
        # a few requests with short drafts in the framework's own precision, distance bias
        _tree("tree_r8_n5_f32", 8, 2000, 5, 16, 16, 64, "f32", 16, 0.0, True),
        # a full serving batch with drafted trees over ragged contexts, capped scores
        _tree("tree_r48_n16_bf16", 48, 8192, 16, 32, 8, 128, "bf16", 64, 30.0, False),
        # one row of the benchmark decoder's vocabulary
        _sample("sample_n1_v50304_f32", 1, 50304, "f32", True, True, False, False),
        # a batch with masked-out tokens, min-p and some greedy rows, odd vocabulary
        _sample("sample_n37_v32003_f16", 37, 32003, "f16", False, False, True, True),
        # a large batch over a large vocabulary, nucleus sampling
        _sample("sample_n256_v131072_bf16", 256, 131072, "bf16", True, True, True, False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One more case: any operator and type, sizes spread over their logarithm up to the largest listed."""
    op = rng.choice(("rotary", "rules", "rules", "tree", "tree", "sample"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    head = rng.choice((32, 64, 64, 80, 96, 128, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    if op == "rotary":
        layout = rng.choice(("halves", "interleaved"))
        rot = rng.choice((head, head, head // 2, head // 4))
        c = _rotary("", _log_int(rng, 1, 8000), heads, kv_heads, head, rot - rot % 2, layout, dtype, rng.choice((16, 24, 64)),
                    _log_int(rng, 100, 1 << 20), rng.choice(("plain", "linear", "bands", "ramp")))
    elif op == "rules":
        # fp32 prompts stay at the framework's own sizes
        length = _log_int(rng, 1, 1500 if dtype == "f32" else 5000)
        most = max(1, min(8, int(4 * 2048 * 2048 * 16 / (length * length * heads))))
        c = _rules("", _log_int(rng, 1, most), heads, kv_heads, length, head, dtype, rng.random() < 0.7,
                   rng.choice((0.0, 0.0, 20.0, 50.0)), rng.random() < 0.4, rng.choice((0, 0, 3, 9)), rng.random() < 0.3)
    elif op == "tree":
        longest = _log_int(rng, 1, 8000)
        c = _tree("", _log_int(rng, 1, max(1, min(48, 200000 // longest))), longest, rng.choice((1, 1, 2, 7, 16, 24)), heads,
                  kv_heads, head, dtype, rng.choice((16, 24, 64)), rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.3)
    else:
        vocab = _log_int(rng, 1000, 131072)
        c = _sample("", _log_int(rng, 1, max(1, min(512, 33000000 // vocab))), vocab, dtype, rng.random() < 0.5,
                    rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.4)
    del c["name"]
    return c


# ------------------------------------------------------------------ lengths (of the case, whatever the seed)
def _document_lengths(c):
    """Ragged documents that fill a row of the batch, the first about half of it."""
    n, left, out = c["documents"], c["length"], []
    for i in range(n):
        take = left if i == n - 1 else min(left, max(1, left * 9 // 20 + i) if left else 0)
        out.append(take)
        left -= take
    return out


def _prefix_lengths(c):
    return [c["length"] * (1 + b % 3) // 5 for b in range(c["batch"])]


def _contexts(c):
    """Cached tokens per request: the longest in full, the others ragged, one in sixteen new."""
    rng = random.Random(c["requests"] * 1000003 + c["longest"])
    return [c["longest"] if r == 0 else 0 if r % 16 == 15 else rng.randint(1, c["longest"]) for r in range(c["requests"])]


def _drafts(c):
    return [c["drafts"] if r % 3 == 0 else 1 + (r * 7) % c["drafts"] for r in range(c["requests"])]


def _visible(c):
    """Visible (query, key) pairs of one head, all of the batch."""
    s = c["length"]
    i = np.arange(s)
    total = 0
    for b in range(c["batch"]):
        pre = _prefix_lengths(c)[b] if c["prefix"] else 0
        if c["documents"]:
            start = 0
            for n in _document_lengths(c):
                q = np.arange(start, start + n)
                last = np.maximum(q, min(pre, start + n) - 1) if c["causal"] else np.full(n, start + n - 1)
                total += int((last - start + 1).sum())
                start += n
        else:
            total += int((np.maximum(i, pre - 1) + 1).sum()) if c["causal"] else s * s
    return total


def work(case):
    """Every input read once and every output written once; products of visible pairs only."""
    c = case
    e = torch.finfo(_TYPES[c["dtype"]]).bits // 8
    if c["op"] == "rotary":
        row = (c["heads"] + 2 * c["kv_heads"]) * c["head"]
        turned = (c["heads"] + c["kv_heads"]) * c["rot"]
        return {"bytes": c["tokens"] * (2 * row * e + 16), "flops": 3 * turned * c["tokens"]}
    if c["op"] == "rules":
        rows = c["batch"] * c["length"]
        return {"bytes": rows * c["head"] * 2 * (c["heads"] + c["kv_heads"]) * e, "flops": 4 * c["head"] * c["heads"] * _visible(c)}
    if c["op"] == "tree":
        ctx, n = _contexts(c), _drafts(c)
        cached = sum(a + b for a, b in zip(ctx, n))
        pairs = sum(a * b + b * (b + 1) // 2 for a, b in zip(ctx, n))
        return {"bytes": 2 * c["head"] * e * (cached * c["kv_heads"] + sum(n) * c["heads"]), "flops": 4 * c["head"] * c["heads"] * pairs}
    return {"bytes": c["rows"] * (c["vocab"] * e + 28), "flops": 4 * c["rows"] * c["vocab"]}


# ------------------------------------------------------------------ inputs
def _frequencies(c):
    """Radians per position of each pair, scaled for long contexts, and the factor on both functions."""
    rot, base, factor, length = c["rot"], 10000.0, 8.0, 4096.0
    i = np.arange(rot // 2, dtype=np.float64)
    f, magnitude = base ** (-2.0 * i / rot), 1.0
    if c["scaling"] == "linear":
        f = f / factor
    elif c["scaling"] == "bands":  # few turns over the trained length: stretched; many: kept
        keep = np.clip((length * f / (2 * math.pi) - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        f = f * ((1.0 - keep) / factor + keep)
    elif c["scaling"] == "ramp":  # the same by the pair's index, between 32 turns and one
        at = lambda turns: rot * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        stretch = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        f, magnitude = f * (stretch / factor + 1.0 - stretch), 0.1 * math.log(factor) + 1.0
    return f.astype(np.float32), magnitude


def _slopes(heads, device):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device=device)


def _parents(n, rng):
    """A tree of n drafts as bit masks: each sees itself and what its parent sees."""
    masks = []
    for j in range(n):
        parent = rng.randint(max(0, j - 4), j - 1) if j else -1
        masks.append((masks[parent] if j else 0) | 1 << j)
    return masks


def prepare(case, seed):
    c, device = case, "cuda"
    g = torch.Generator(device=device)
    g.manual_seed(int(seed) * 7919 + 17)
    host = random.Random(int(seed) * 31 + 5)
    t = _TYPES[c["dtype"]]
    randn = lambda *shape: torch.randn(shape, generator=g, device=device).to(t)  # noqa: E731
    s = {"case": c}
    if c["op"] == "rotary":
        n, h, kv, d, page = c["tokens"], c["heads"], c["kv_heads"], c["head"], c["page"]
        qkv = randn(n, (h + 2 * kv) * d)  # one projection: queries, keys and values side by side
        s["q"], s["k"], s["v"] = (x.unflatten(-1, (-1, d)) for x in qkv.split((h * d, kv * d, kv * d), -1))
        f, s["magnitude"] = _frequencies(c)
        s["frequencies"] = torch.from_numpy(f).to(device)
        last = max(c["longest"], n)
        s["positions"] = torch.arange(n, device=device) + host.randint(0, last - n)
        pages = -(-n // page) + 3
        order = torch.randperm(pages, generator=g, device=device)
        at = torch.arange(n, device=device) + host.randint(0, page - 1)
        s["slots"] = order[at // page] * page + at % page
        s["q_out"] = torch.empty((n, h, d), dtype=t, device=device)
        s["k_cache"], s["v_cache"] = (torch.zeros((pages, page, kv, d), dtype=t, device=device) for _ in range(2))
    elif c["op"] == "rules":
        b, h, kv, n, d = c["batch"], c["heads"], c["kv_heads"], c["length"], c["head"]
        s["q"], s["k"], s["v"] = (randn(b, n, x, d).transpose(1, 2) for x in (h, kv, kv))  # heads are views of the rows
        if c["cap"]:
            s["q"] = (s["q"] * 3).contiguous().transpose(1, 2).contiguous().transpose(1, 2)  # scores that reach the cap's bend
        s["out"] = torch.empty((b, n, h, d), dtype=t, device=device).transpose(1, 2)
        s["slopes"] = _slopes(h, device) if c["bias"] else None
        s["prefix"] = torch.tensor(_prefix_lengths(c), dtype=torch.int32, device=device) if c["prefix"] else None
        s["documents"] = None
        if c["documents"]:
            lengths = torch.tensor(_document_lengths(c))
            s["documents"] = torch.repeat_interleave(torch.arange(c["documents"]), lengths).to(torch.int32).expand(b, n).contiguous().to(device)
    elif c["op"] == "tree":
        h, kv, d, page = c["heads"], c["kv_heads"], c["head"], c["page"]
        ctx, n = _contexts(c), _drafts(c)
        need = [-(-(a + b) // page) for a, b in zip(ctx, n)]
        order = list(range(sum(need) + 2))
        host.shuffle(order)
        table = np.zeros((c["requests"], max(need)), np.int32)
        at = 0
        for r, k in enumerate(need):
            table[r, :k] = order[at:at + k]
            at += k
        s["block_table"] = torch.from_numpy(table).to(device)
        s["context"] = torch.tensor(ctx, dtype=torch.int32, device=device)
        s["query_start"] = torch.tensor(np.concatenate([[0], np.cumsum(n)]).tolist(), dtype=torch.int32, device=device)
        s["tree"] = torch.tensor(sum((_parents(k, host) for k in n), []), dtype=torch.int64, device=device) if c["drafts"] > 1 else None
        s["q"] = randn(sum(n), h, d)
        s["k_cache"], s["v_cache"] = randn(len(order), page, kv, d), randn(len(order), page, kv, d)
        s["out"] = torch.empty((sum(n), h, d), dtype=t, device=device)
        s["slopes"] = _slopes(h, device) if c["bias"] else None
        s["workspace"] = torch.empty(32 << 20, dtype=torch.uint8, device=device)
        s["most"], s["total"] = max(n), max(a + b for a, b in zip(ctx, n))
    else:
        n, v = c["rows"], c["vocab"]
        z = torch.randn((n, v), generator=g, device=device) * 2.5
        likely = torch.randint(0, v, (n, 12), generator=g, device=device)
        z.scatter_add_(1, likely, torch.rand((n, 12), generator=g, device=device) * 9)  # what the context calls for
        if c["masked"]:  # a grammar rules tokens out
            z.masked_fill_(torch.rand((n, v), generator=g, device=device) < 0.3, -math.inf)
        s["logits"] = z.to(t)
        unit = lambda: torch.rand(n, generator=g, device=device)  # noqa: E731
        s["uniform"] = unit()
        warm = 0.5 + unit()
        s["temperature"] = torch.where(unit() < 0.1, torch.zeros_like(warm), warm)  # some rows are greedy
        s["top_k"] = torch.randint(1, 200, (n,), generator=g, device=device, dtype=torch.int32) if c["top_k"] else None
        if c["top_k"] and n > 1:  # every other row is without
            s["top_k"][1::2] = 0
        s["top_p"] = 0.7 + 0.3 * unit() if c["top_p"] else None
        s["min_p"] = 0.1 * unit() if c["min_p"] else None
        s["tokens"] = torch.empty(n, dtype=torch.int64, device=device)
        s["probabilities"] = torch.empty(n, dtype=torch.float32, device=device)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["frequencies"].double()
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x):
        x, rot = x.float(), c["rot"]
        if c["layout"] == "halves":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((y, x[..., rot:]), -1)

    dtype = s["q"].dtype
    s["q_out"].copy_(turned(s["q"]).to(dtype))
    s["k_cache"].flatten(0, 1)[s["slots"]] = turned(s["k"]).to(dtype)
    s["v_cache"].flatten(0, 1)[s["slots"]] = s["v"]
    return s["q_out"], s["k_cache"], s["v_cache"]


def _weighted(scores, visible, v):
    """Softmax over the visible keys times the values; rows that see nothing are zero."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)


def _plain_rules(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    q, k, v = s["q"].float(), s["k"].float().repeat_interleave(group, 1), s["v"].float().repeat_interleave(group, 1)
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(c["head"])
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    at = torch.arange(c["length"], device=q.device)
    if s["slopes"] is not None:
        scores = scores - s["slopes"][:, None, None] * (at[:, None] - at).abs()
    visible = torch.ones((1, 1, c["length"], c["length"]), dtype=torch.bool, device=q.device)
    if c["causal"]:
        visible = (at <= at[:, None])[None, None]
        if s["prefix"] is not None:
            visible = visible | (at < s["prefix"][:, None, None, None])
    if s["documents"] is not None:
        visible = visible & (s["documents"][:, None, :, None] == s["documents"][:, None, None, :])
    s["out"].copy_(_weighted(scores, visible, v).to(s["q"].dtype))
    return s["out"]


def _plain_tree(s):
    c = s["case"]
    r, n, total, group = c["requests"], s["most"], s["total"], c["heads"] // c["kv_heads"]
    device = s["q"].device
    key = torch.arange(total, device=device)
    page = s["block_table"].long()[:, (key // c["page"]).clamp(max=s["block_table"].shape[1] - 1)]  # [requests, keys]
    k, v = (x[page, key % c["page"]].float().transpose(1, 2).repeat_interleave(group, 1) for x in (s["k_cache"], s["v_cache"]))
    first, count = s["query_start"][:-1].long(), s["query_start"].diff().long()
    j = torch.arange(n, device=device)
    row = (first[:, None] + j).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().transpose(1, 2)  # [requests, heads, drafts, head]
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(c["head"])
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    seen = (s["tree"][row] if s["tree"] is not None else ((2 << j) - 1).expand(r, n))  # bit masks over the drafts
    context = s["context"].long()[:, None]
    draft = key - context  # [requests, keys]: which draft a key is
    bit = (seen[:, :, None] >> draft.clamp(0, 62)[:, None, :] & 1).bool()
    visible = (draft < 0)[:, None, :] | bit & ((draft >= 0) & (draft < count[:, None]))[:, None, :]
    if s["slopes"] is not None:  # a draft's position is its depth in the tree
        depth = (seen[:, :, None] >> j & 1).sum(-1) - 1
        q_at = context + depth
        k_at = torch.where(draft < 0, key, context + depth.gather(1, draft.clamp(0, n - 1)))
        scores = scores - s["slopes"][:, None, None] * (q_at[:, :, None] - k_at[:, None, :]).abs()[:, None]
    out = _weighted(scores, visible[:, None], v).transpose(1, 2)
    s["out"].copy_(out[j < count[:, None]].to(s["q"].dtype))
    return s["out"]


def _plain_sample(s):
    z = s["logits"].double()
    rows, vocab = z.shape
    z = torch.where(z.isnan(), torch.full_like(z, -math.inf), z)
    warm = s["temperature"].double()[:, None]
    greedy = ~(warm > 0)
    top = z.amax(-1, keepdim=True)
    w = torch.exp((z - top) / torch.where(greedy, torch.ones_like(warm), warm))
    w, order = torch.sort(w, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    rank = torch.arange(vocab, device=z.device)
    kept = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        kept &= (rank < k) | (k <= 0)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        inside = w * kept
        before = inside.cumsum(-1) - inside
        kept &= (before < p * inside.sum(-1, keepdim=True)) | (rank == 0) | (p >= 1)
    if s["min_p"] is not None:
        kept &= w >= s["min_p"].double().clamp(max=1)[:, None]
    kept &= ~greedy | (rank == 0)
    w = torch.zeros_like(w).scatter_(-1, order, w * kept)  # back to the vocabulary's order
    upto = w.cumsum(-1)
    total = upto[:, -1:]
    token = (upto <= s["uniform"].double()[:, None] * total).sum(-1).clamp(max=vocab - 1)
    s["tokens"].copy_(token)
    s["probabilities"].copy_((w.gather(-1, token[:, None]) / total)[:, 0].float())
    return s["tokens"], s["probabilities"]


# ------------------------------------------------------------------ the framework's calls
def _own_rotary(s, cabi, stream):
    layout = cabi.ROTARY_HALVES if s["case"]["layout"] == "halves" else cabi.ROTARY_INTERLEAVED
    cabi.rotary_positions(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["frequencies"], s["q_out"], s["k_cache"],
                          s["v_cache"], magnitude=s["magnitude"], layout=layout, stream=stream)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _own_rules(s, cabi, stream):
    c = s["case"]
    cabi.attention_rules(s["q"], s["k"], s["v"], s["out"], math.sqrt(c["head"]), cap=c["cap"], causal=c["causal"],
                         slopes=s["slopes"], prefix=s["prefix"], q_documents=s["documents"], k_documents=s["documents"], stream=stream)
    return s["out"]


def _own_tree(s, cabi, stream):
    c = s["case"]
    cabi.attention_tree(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["context"], s["query_start"], s["tree"], s["out"],
                        s["workspace"], math.sqrt(c["head"]), cap=c["cap"], slopes=s["slopes"], stream=stream)
    return s["out"]


def _own_sample(s, cabi, stream):
    cabi.sample(s["logits"], s["uniform"], s["tokens"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                min_p=s["min_p"], probabilities=s["probabilities"], stream=stream)
    return s["tokens"], s["probabilities"]


_PLAIN = {"rotary": _plain_rotary, "rules": _plain_rules, "tree": _plain_tree, "sample": _plain_sample}
_OWN = {"rotary": _own_rotary, "rules": _own_rules, "tree": _own_tree, "sample": _own_sample}


def run(state):
    if own:
        from fluidml_b200 import cabi
        return _OWN[state["case"]["op"]](state, cabi, torch.cuda.current_stream().cuda_stream)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rotary(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    turn = torch.polar(torch.full((c["tokens"], half), float(s["magnitude"]), dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["frequencies"].double()))[:, None, :]
    first = torch.arange(half, device="cuda") if c["layout"] == "halves" else torch.arange(0, rot, 2, device="cuda")
    second = first + (half if c["layout"] == "halves" else 1)

    def turned(x):
        x = x.double().clone()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    caches = []
    for x in (turned(s["k"]), s["v"].double()):
        cache = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device="cuda")
        cache[s["slots"] // c["page"], s["slots"] % c["page"]] = x
        caches.append(cache)
    return (turned(s["q"]), *caches)


def _exact_row(q, k, v, bias, visible, divisor, cap):
    """One head in 64 bits: q [n, d], k, v [m, d], bias and visible [n, m] (bias may be None)."""
    x = q.double() @ k.double().T / divisor
    if cap:
        x = cap * (1 - 2 / (torch.exp(2 * x / cap) + 1))
    if bias is not None:
        x = x + bias
    x = torch.where(visible, x, torch.tensor(-math.inf, dtype=torch.float64, device=x.device))
    lse = torch.logsumexp(x, -1, keepdim=True)
    return torch.where(lse > -math.inf, torch.exp(x - lse), torch.zeros_like(x)) @ v.double()


def _exact_rules(s):
    c = s["case"]
    n, d, group = c["length"], c["head"], c["heads"] // c["kv_heads"]
    i = torch.arange(n, device="cuda").double()
    out = torch.empty((c["batch"], c["heads"], n, d), dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        visible = i[None, :] <= i[:, None] if c["causal"] else torch.ones((n, n), dtype=torch.bool, device="cuda")
        if s["prefix"] is not None and c["causal"]:
            visible = visible | (i < s["prefix"][b].double())[None, :]
        if s["documents"] is not None:
            visible = visible & (s["documents"][b][:, None] == s["documents"][b][None, :])
        for h in range(c["heads"]):
            bias = -s["slopes"][h].double() * (i[:, None] - i[None, :]).abs() if s["slopes"] is not None else None
            out[b, h] = _exact_row(s["q"][b, h], s["k"][b, h // group], s["v"][b, h // group], bias, visible, math.sqrt(d), c["cap"])
    return out


def _exact_tree(s):
    c = s["case"]
    group, start = c["heads"] // c["kv_heads"], s["query_start"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, ctx in enumerate(s["context"].tolist()):
        a, b = start[r], start[r + 1]
        n = b - a
        pages = s["block_table"][r].long()
        k, v = (x[pages].flatten(0, 1)[:ctx + n] for x in (s["k_cache"], s["v_cache"]))
        seen = s["tree"][a:b].tolist() if s["tree"] is not None else [(2 << j) - 1 for j in range(n)]
        tree = torch.tensor([[m >> j & 1 for j in range(n)] for m in seen], dtype=torch.bool, device="cuda").reshape(n, n)
        visible = torch.cat((torch.ones((n, ctx), dtype=torch.bool, device="cuda"), tree), 1)
        depth = tree.sum(1).double() - 1
        at = torch.cat((torch.arange(ctx, device="cuda").double(), ctx + depth))
        for h in range(c["heads"]):
            bias = -s["slopes"][h].double() * ((ctx + depth)[:, None] - at).abs() if s["slopes"] is not None else None
            out[a:b, h] = _exact_row(s["q"][a:b, h], k[:, h // group], v[:, h // group], bias, visible, math.sqrt(c["head"]), c["cap"])
    return out


def _exact_sample(s):
    z, u, warm = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy(), s["temperature"].double().cpu().numpy()
    given = {k: s[k].cpu().numpy() if s[k] is not None else None for k in ("top_k", "top_p", "min_p")}
    tokens, probabilities = [], []
    for r in range(z.shape[0]):
        order = np.argsort(-z[r], kind="stable")
        if not warm[r] > 0:
            tokens.append(int(order[0]))
            probabilities.append(1.0)
            continue
        order = order[z[r][order] > -np.inf]
        if given["top_k"] is not None and given["top_k"][r] > 0:
            order = order[:given["top_k"][r]]
        w = np.exp((z[r][order] - z[r][order[0]]) / warm[r])
        if given["top_p"] is not None and given["top_p"][r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            n = max(1, int((before < float(given["top_p"][r]) * w.sum()).sum()))
            order, w = order[:n], w[:n]
        if given["min_p"] is not None:
            order, w = order[w >= min(float(given["min_p"][r]), 1.0)], w[w >= min(float(given["min_p"][r]), 1.0)]
        back = np.argsort(order)
        order, w = order[back], w[back]
        at = min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), len(w) - 1)
        tokens.append(int(order[at]))
        probabilities.append(float(w[at] / w.sum()))
    return torch.tensor(tokens), torch.tensor(probabilities, dtype=torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "rules": _exact_rules, "tree": _exact_tree, "sample": _exact_sample}[case["op"]](s)
