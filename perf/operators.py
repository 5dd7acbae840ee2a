"""Operators of a verification step: what is measured, and their plain forms.

A decode step that checks drafted tokens runs one forward over a small tree of
tokens for each request. Three operators carry what a plain decode step does
not have: the per-head norms and the rotation of queries and keys
(``qk_norm_rope``), the attention of the tree's nodes over the selected cache
rows and over each other (``attend_tree``), and the log probabilities, entropy
and alternatives at every node (``token_logprobs``).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "nano-hisparse_b200")
_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_DEVICE = "cuda:0"


# ---- the cases ---------------------------------------------------------------------------
def _norm_rope(name, tokens, q_heads, kv_heads, head_dim, dtype, start, prompt):
    return {"name": name, "op": "qk_norm_rope", "tokens": tokens, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "start": start,
            "prompt": prompt}


def _logprobs(name, rows, vocab, given, top, dtype, masked):
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "given": given,
            "top": top, "dtype": dtype, "masked": masked}


def _tree(name, batch, nodes, q_heads, kv_heads, head_dim, page_size, rows, dtype):
    return {"name": name, "op": "attend_tree", "batch": batch, "nodes": nodes,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "page_size": page_size, "rows": rows, "dtype": dtype}


def listed():
    return [
        # one decode token of the small fp32 decoder (8/2 heads of 32): launch latency
        _norm_rope("rope_decode_1", 1, 8, 2, 32, "float32", 160, False),
        # a verification step of 16 requests, 8 nodes each, at 32k context
        _norm_rope("rope_verify_128", 128, 32, 8, 128, "bfloat16", 32768, False),
        # an odd prompt piece near one million tokens (28/4 heads), fp16
        _norm_rope("rope_piece_4099", 4099, 28, 4, 128, "float16", 1044477, True),
        # a whole 32k prompt
        _norm_rope("rope_prompt_32768", 32768, 32, 8, 128, "bfloat16", 0, True),
        # the small fp32 decoder's step: three requests
        _logprobs("logprobs_decode_3", 3, 1024, 1, 4, "float32", False),
        # 16 requests of one token each, 20 alternatives
        _logprobs("logprobs_decode_16", 16, 128256, 1, 20, "bfloat16", False),
        # a tree of 63 nodes, up to four drafted children scored at each, part of the
        # vocabulary ruled out
        _logprobs("logprobs_tree_63", 63, 128256, 4, 1, "bfloat16", True),
        # scoring a prompt of 2,048 tokens with five alternatives, fp32 logits
        _logprobs("logprobs_prompt_2048", 2048, 128256, 1, 5, "float32", False),
        # the small fp32 decoder: three requests, trees of five nodes over 160 rows
        _tree("tree_small_fp32", 3, 5, 8, 2, 32, 16, 160, "float32"),
        # 16 requests, 8 nodes, the 2,048-row Quest budget
        _tree("tree_budget_2048", 16, 8, 32, 8, 128, 16, 2048, "bfloat16"),
        # one long request, 63 nodes, the 8,192-row budget in pages of 64 (28/4 heads)
        _tree("tree_long_8192", 1, 63, 28, 4, 128, 64, 8192, "bfloat16"),
        # full history at 32k: 8 requests, 32 nodes
        _tree("tree_full_32768", 8, 32, 32, 8, 128, 16, 32768, "bfloat16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_HEADS = [(8, 2, 32), (32, 8, 128), (28, 4, 128), (16, 16, 64), (10, 2, 80), (12, 1, 256)]


def draw(rng):
    op = rng.choice(["qk_norm_rope", "token_logprobs", "attend_tree"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    hq, hkv, d = rng.choice(_HEADS)
    if op == "qk_norm_rope":
        limit = 32768 * 40 * 128 // ((hq + hkv) * d * (2 if dtype == "float32" else 1))
        prompt = rng.random() < 0.5
        tokens = _spread(rng, 1, min(32768, limit) if prompt else 512)
        case = _norm_rope("", tokens, hq, hkv, d, dtype, rng.randrange(1 << 20), prompt)
    elif op == "token_logprobs":
        vocab = _spread(rng, 256, 128256)
        rows = _spread(rng, 1, 2048)
        case = _logprobs("", rows, vocab, rng.choice([1, 1, 2, 4]), rng.choice([0, 1, 5, 20]),
                         dtype, rng.random() < 0.3)
    else:
        batch, nodes = _spread(rng, 1, 16), _spread(rng, 1, 64)
        # at most the largest listed case's products, an eighth of them in fp32
        budget = 8 * 32 * 32 * 128 * 32768 // (8 if dtype == "float32" else 1)
        limit = budget // (batch * nodes * hq * d)
        rows = _spread(rng, 1, max(1, min(32768, limit, 8 * 32768 * 1024 // (batch * hkv * d))))
        case = _tree("", batch, nodes, hq, hkv, d, rng.choice([16, 64, 12]), rows, dtype)
    del case["name"]
    return case


# ---- ragged sizes, from the case alone ----------------------------------------------------
def _row_counts(case):
    """Rows each request holds: the longest first, the shortest three quarters of it."""
    b, n = case["batch"], case["rows"]
    return [n - i * n // (4 * b) for i in range(b)]


def _node_counts(case):
    """Nodes of each request's tree: up to two fewer than the widest."""
    return [max(1, case["nodes"] - i % 3) for i in range(case["batch"])]


def _parents(nodes):
    """A drafted tree: node 0 is the pending token, every second node extends the
    chain before it, the others branch off near the root."""
    return [-1] + [t - 1 if t % 2 else (t - 1) // 4 for t in range(1, nodes)]


def _ancestors(nodes):
    masks = []
    for t, p in enumerate(_parents(nodes)):
        masks.append((masks[p] if p >= 0 else 0) | 1 << t)
    return masks


# ---- inputs -------------------------------------------------------------------------------
def prepare(case, seed):
    if own and _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        x = torch.empty(shape, dtype=dtype, device=_DEVICE)
        return x.normal_(0.0, scale, generator=gen)

    state = {"case": case}
    if case["op"] == "qk_norm_rope":
        n, hq, hkv, d = (case[k] for k in ("tokens", "q_heads", "kv_heads", "head_dim"))
        # the fused projection's output: queries, keys and values side by side
        fused = normal(n, (hq + 2 * hkv) * d)
        state["query"] = fused[:, :hq * d].view(n, hq, d)
        state["key"] = fused[:, hq * d:(hq + hkv) * d].view(n, hkv, d)
        if case["prompt"]:  # consecutive positions
            state["positions"] = case["start"] + torch.arange(n, device=_DEVICE)
        else:  # requests of different lengths
            state["positions"] = torch.randint(0, case["start"] + 1, (n,), generator=gen,
                                               device=_DEVICE)
        state["query_weight"] = 1 + normal(d, scale=0.1, dtype=torch.float32).to(dtype)
        state["key_weight"] = 1 + normal(d, scale=0.1, dtype=torch.float32).to(dtype)
        exponent = torch.arange(0, d, 2, dtype=torch.float64, device=_DEVICE) / d
        state["inv_freq"] = 10000.0 ** -exponent
    elif case["op"] == "token_logprobs":
        n, v = case["rows"], case["vocab"]
        logits = normal(n, v, scale=3.0)
        if case["masked"]:  # every third token ruled out
            logits[:, 1::3] = -math.inf
        tokens = torch.randint(0, (v + 2) // 3, (n, case["given"]), generator=gen,
                               device=_DEVICE) * 3
        tokens.clamp_(max=(v - 1) // 3 * 3)
        if case["given"] > 1:  # nodes with fewer children than the widest
            tokens[1::2, -1] = -1
        state["logits"], state["tokens"] = logits, tokens
    else:
        b, t, hq, hkv, d, p = (case[k] for k in ("batch", "nodes", "q_heads", "kv_heads",
                                                 "head_dim", "page_size"))
        width = case["rows"]
        pages = -(-width // p)
        blocks = b * pages + 7
        state["pool"] = normal(blocks, 2, p, hkv, d)
        order = torch.randperm(blocks, generator=gen, device=_DEVICE)[:b * pages].view(b, pages)
        rows = (order[:, :, None] * p + torch.arange(p, device=_DEVICE)).view(b, pages * p)
        rows = rows[:, :width].contiguous()
        counts = torch.tensor(_row_counts(case), dtype=torch.int32, device=_DEVICE)
        column = torch.arange(width, device=_DEVICE)
        rows[column[None, :] >= counts[:, None]] = -1
        state["rows"], state["counts"] = rows, counts
        # one fused projection's output, as the queries, keys and values of the nodes
        fused = normal(b, t, (hq + 2 * hkv) * d)
        state["query"] = fused[..., :hq * d].unflatten(-1, (hq, d))
        state["query"].mul_(1.5)
        state["key"] = fused[..., hq * d:(hq + hkv) * d].unflatten(-1, (hkv, d))
        state["value"] = fused[..., (hq + hkv) * d:].unflatten(-1, (hkv, d))
        masks = [m - (1 << 64) if m >> 63 else m for m in _ancestors(t)]
        state["mask"] = torch.tensor([masks] * b, dtype=torch.int64, device=_DEVICE)
        state["nodes"] = torch.tensor(_node_counts(case), dtype=torch.int32, device=_DEVICE)
        if own:
            from hisparse_b200 import CacheConfig

            state["config"] = CacheConfig(gpu_pages=blocks, page_size=p, kv_heads=hkv,
                                          head_dim=d, device=_DEVICE, dtype=dtype)
    return state


# ---- one pass -----------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        import hisparse_b200 as hs

        if op == "qk_norm_rope":
            return hs.qk_norm_rope(state["query"], state["key"], state["positions"],
                                   state["inv_freq"], state["query_weight"],
                                   state["key_weight"], eps=1e-6)
        if op == "token_logprobs":
            return tuple(hs.token_logprobs(state["logits"], state["tokens"],
                                           top=state["case"]["top"]))
        return hs.attend_tree(state["query"], state["key"], state["value"], state["mask"],
                              state["pool"], state["rows"], state["config"],
                              counts=state["counts"], nodes=state["nodes"])
    if op == "qk_norm_rope":
        return _plain_norm_rope(state)
    if op == "token_logprobs":
        return _plain_logprobs(state)
    return _plain_tree(state)


def _plain_norm_rope(state):
    angles = state["positions"].double()[:, None] * state["inv_freq"][None, :]
    cosine, sine = angles.cos().float()[:, None, :], angles.sin().float()[:, None, :]
    out = []
    for x, weight in ((state["query"], state["query_weight"]),
                      (state["key"], state["key_weight"])):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
        a, b = y.chunk(2, -1)
        out.append(torch.cat((a * cosine - b * sine, b * cosine + a * sine), -1).to(x.dtype))
    return tuple(out)


def _plain_logprobs(state):
    x, tokens, top = state["logits"].float(), state["tokens"], state["case"]["top"]
    largest = x.amax(-1, keepdim=True)
    weights = torch.exp(x - largest)
    total = weights.sum(-1, keepdim=True)
    lse = largest + torch.log(total)
    given = torch.gather(x, 1, tokens.clamp(min=0)) - lse
    given = torch.where(tokens >= 0, given, torch.zeros_like(given))
    logp = x - lse
    entropy = -torch.where(weights > 0, weights * logp, torch.zeros_like(logp)).sum(-1)
    entropy = entropy / total[:, 0]
    values, indices = torch.sort(x, dim=-1, descending=True, stable=True)
    return given, entropy, values[:, :top] - lse, indices[:, :top].contiguous()


def _plain_tree(state):
    case, pool, rows = state["case"], state["pool"], state["rows"]
    q, k, v = state["query"].float(), state["key"].float(), state["value"].float()
    b, t, hq, d = q.shape
    p, hkv = case["page_size"], case["kv_heads"]
    groups, width = hq // hkv, rows.shape[1]
    column = torch.arange(width, device=rows.device)
    valid = (rows >= 0) & (column[None, :] < state["counts"][:, None])
    block, within = rows.clamp(min=0) // p, rows.clamp(min=0) % p
    keys = torch.cat((pool[block, 0, within].float(), k), 1)      # [b, width + t, hkv, d]
    values = torch.cat((pool[block, 1, within].float(), v), 1)
    node = torch.arange(t, device=rows.device)
    real = node[None, :] < state["nodes"][:, None]                # [b, t]
    sees = (state["mask"][:, :, None] >> node) & 1 == 1           # [b, t, t]
    sees = sees & real[:, None, :]
    visible = torch.cat((valid[:, None, :].expand(b, t, width), sees), -1)
    q = q.view(b, t, hkv, groups, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * groups, d)
    scores = torch.matmul(q, keys.permute(0, 2, 3, 1)) / math.sqrt(d)
    scores = scores.view(b, hkv, t, groups, width + t)
    scores = scores.masked_fill(~visible[:, None, :, None, :], -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(b, hkv, t * groups, width + t), values.permute(0, 2, 1, 3))
    out = out.view(b, hkv, t, groups, d) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(b, t, hq, d)
    out = torch.where(real[:, :, None, None], out, torch.zeros_like(out))
    return out.to(state["query"].dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "qk_norm_rope":
        return tuple(_exact_norm_rope(state, which) for which in ("query", "key"))
    if case["op"] == "token_logprobs":
        return _exact_logprobs(state)
    return _exact_tree(state)


def _exact_norm_rope(state, which):
    x, weight = state[which].double(), state[which + "_weight"].double()
    half = x.shape[-1] // 2
    size = (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt()
    y = x / size * weight
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       torch.outer(state["positions"].double(), state["inv_freq"]))
    rotated = torch.complex(y[..., :half], y[..., half:]) * turn[:, None, :]
    return torch.cat((rotated.real, rotated.imag), -1)


def _exact_logprobs(state):
    top, parts = state["case"]["top"], []
    vocab = state["logits"].shape[1]
    backwards = torch.arange(vocab - 1, -1, -1, device=_DEVICE)
    step = max(1, (1 << 25) // vocab)
    for first in range(0, state["logits"].shape[0], step):
        x = state["logits"][first:first + step].double()
        tokens = state["tokens"][first:first + step]
        logp = torch.log_softmax(x, -1)
        p = logp.exp()
        entropy = -torch.special.xlogy(p, p).sum(-1)
        given = logp.gather(1, tokens.clamp(min=0)).masked_fill(tokens < 0, 0.0)
        # one whole number for each entry: its value's order, then the lower index first
        bits = (x.float() + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        best = (order * vocab + backwards).topk(top, -1).values
        index = vocab - 1 - best.remainder(vocab)
        parts.append((given, entropy, logp.gather(1, index), index))
    return tuple(torch.cat(column) for column in zip(*parts))


def _exact_tree(state):
    case, pool = state["case"], state["pool"]
    p, hkv, t, d = case["page_size"], case["kv_heads"], case["nodes"], case["head_dim"]
    groups = case["q_heads"] // hkv
    out = torch.zeros((case["batch"], t, case["q_heads"], d), dtype=torch.float64,
                      device=pool.device)
    for b, (count, nodes) in enumerate(zip(_row_counts(case), _node_counts(case))):
        rows = state["rows"][b, :count]
        pairs = torch.stack([pool[rows // p, i, rows % p] for i in (0, 1)], 1)
        bias = torch.zeros((nodes, count + nodes), dtype=torch.float64)
        for i, seen in enumerate(_ancestors(t)[:nodes]):
            for j in range(nodes):
                if not seen >> j & 1:
                    bias[i, count + j] = -math.inf
        bias = bias.to(pool.device)
        for h in range(hkv):
            keys = torch.cat((pairs[:, 0, h], state["key"][b, :nodes, h])).double()
            values = torch.cat((pairs[:, 1, h], state["value"][b, :nodes, h])).double()
            for g in range(h * groups, (h + 1) * groups):
                q = state["query"][b, :nodes, g].double()
                probabilities = torch.softmax(q @ keys.T / d ** 0.5 + bias, -1)
                out[b, :nodes, g] = probabilities @ values
    return out


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "qk_norm_rope":
        n, d = case["tokens"], case["head_dim"]
        elements = n * (case["q_heads"] + case["kv_heads"]) * d
        return {"bytes": 2 * elements * size + n * 8 + 2 * d * size + d // 2 * 8,
                "flops": 10 * elements}
    if case["op"] == "token_logprobs":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * (v * size + case["given"] * 12 + 4 + case["top"] * 12),
                "flops": 6 * n * v}
    hq, hkv, d, t = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "nodes"))
    counts, nodes = _row_counts(case), _node_counts(case)
    moved = sum(c * (2 * hkv * d * size + 8) for c in counts)
    moved += sum(n * (hq + 2 * hkv) * d * size for n in nodes)
    moved += case["batch"] * t * (hq * d * size + 8) + case["batch"] * 8
    pairs = sum(n * c + sum(bin(m).count("1") for m in _ancestors(t)[:n])
                for c, n in zip(counts, nodes))
    return {"bytes": moved, "flops": 4 * pairs * hq * d}
