"""Drafted decoding in 16-bit types, part by part: the attention of every drafted layer, the
rows that it appends, the scores and the choice of every emitted token, and the whole forward
against a dense one in fp64.

u is half a step of the type (bf16 2^-8, fp16 2^-11), f = 2^-24 half a step of fp32.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_verify_engine import (DEV, MODEL, PROMPTS, Oracle, add_requests, dense_logits,
                                    make_engine, no_flags, plain_run)
from test_gpu_verify_ops import F, half_step, tree_check

pytestmark = pytest.mark.gpu


class Watched:
    """A drafted engine whose steps leave what went through them: the trees, the inputs and
    the result of every layer_tree call and the logits of every forward."""

    def __init__(self, engine, monkeypatch):
        from hisparse_b200.batched import DecodeBatch

        self.engine, self.trees, self.layers, self.logits = engine, {}, [], []
        draft, head, layer_tree = engine._draft, engine.model.head, DecodeBatch.layer_tree

        def watched_draft(request):
            self.trees[request.request_id] = draft(request)
            return self.trees[request.request_id]

        def watched_head(x):
            self.logits.append(head(x))
            return self.logits[-1]

        def watched_layer(batch, layer, query, key, value, *rest):
            out = layer_tree(batch, layer, query, key, value, *rest)
            self.layers.append((batch.request_ids, query, key, value, out))
            return out

        monkeypatch.setattr(engine, "_draft", watched_draft)
        monkeypatch.setattr(engine.model, "head", watched_head)
        monkeypatch.setattr(DecodeBatch, "layer_tree", watched_layer)

    def stored(self, request_id, layer):
        """The K/V rows of a request in the host store, [length, 2, Hkv, D]."""
        cache = self.engine.cache
        blocks = cache.requests[request_id].host[layer]
        rows = cache.host[torch.from_numpy(blocks)].transpose(1, 2).flatten(0, 1)
        return rows[:cache.length(request_id)].clone()

    def step(self):
        engine = self.engine
        engine.cache.rows.synchronize()
        self.trees, self.layers, self.logits = {}, [], []
        emitted = engine.step()
        engine.cache.rows.synchronize()
        return emitted


def paths_of(tree):
    """The nodes that each node of a turn sees (node 0 is the last emitted token)."""
    out = [[0]]
    for t, (_, parent) in enumerate(tree, 1):
        out.append(out[parent + 1] + [t])
    return out


def walk(tree, logits, eos, left):
    """(tokens, nodes) of the path that the logits' maxima take through a tree."""
    best, tokens, nodes = logits.float().argmax(-1).tolist(), [], []
    node = 0
    while node is not None:
        nodes.append(node)
        tokens.append(best[node])
        if tokens[-1] == eos or len(tokens) == left:
            break
        node = next((t for t, (token, parent) in enumerate(tree, 1)
                     if parent + 1 == node and token == tokens[-1]), None)
    return tokens, nodes


def check_scores(scores, rows):
    """Scores against the logits that they were read from: the bounds of token_logprobs."""
    logp = torch.log_softmax(rows.double().cpu(), -1)
    sums = (logp.shape[1] / 128 + 64) * F
    for score, row in zip(scores, logp, strict=True):
        want, order = row.sort(descending=True, stable=True)
        assert [t for t, _ in score.top] == order[:len(score.top)].tolist()
        for (_, have), lp in zip(score.top, want):
            assert abs(have - lp.item()) < sums + 4 * F * abs(lp.item())
        assert abs(score.logprob - want[0].item()) < sums + 4 * F * abs(want[0].item())
        entropy = -(row.exp() * row).sum().item()
        assert abs(score.entropy - entropy) < 2 * sums * (1 + math.log(len(row)))


def check_attention(watched, history):
    """Every layer_tree call over the history that the store held before the step and over
    each node's own path, in fp64 within attend_tree's bound."""
    for layer, (ids, q, k, v, out) in enumerate(watched.layers):
        rows, at = torch.full((len(ids), max(len(history[r][layer]) for r in ids)), -1), 0
        for i, r in enumerate(ids):
            n = len(history[r][layer])
            rows[i, :n], at = at + torch.arange(n), at + n
        pool = torch.cat([history[r][layer] for r in ids])[:, :, None]  # pages of one row
        masks = torch.zeros(q.shape[:2], dtype=torch.int64)
        nodes = torch.zeros(len(ids), dtype=torch.int32)
        for i, r in enumerate(ids):
            for t, path in enumerate(paths_of(watched.trees[r])):
                masks[i, t], nodes[i] = sum(1 << j for j in path), t + 1
        tree_check(out, (q, k, v), masks, pool, rows, None, nodes)


def first_layer_rows(weights, tokens, positions):
    """(K and V rows [n, 2, Hkv, D] of layer 0 in fp64, a bound on the engine's error). The
    norm rounds twice, (2 u + u^2 + 40 f) |h|; the projection adds 132 f and, where its parts
    are joined in the 16-bit type, two more roundings, so 5 u of S = sum |h| |W| + |b| covers
    it. Without head norms cos, sin, the products and their sum round: 3.1 u (|a| + |b|), and
    the fp32 angle is off by f of at most 200 rad, twice. With them the norm of a row off by
    B is off by B / sqrt(D) at most, and the result rounds once."""
    cfg = weights.config
    u, d, hkv = half_step(weights.dtype), cfg.head_dim, cfg.num_key_value_heads
    state = {k: t.double() for k, t in weights.state_dict().items()}
    base = "model.layers.0."
    x = state["model.embed_tokens.weight"][torch.tensor(tokens)]
    h = x / (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt()
    h = h * state[base + "input_layernorm.weight"]
    plain, bound = [], []
    for m in "kv":
        w, b = (state[base + f"self_attn.{m}_proj.{n}"] for n in ("weight", "bias"))
        plain.append((h @ w.t() + b).view(len(tokens), hkv, d))
        bound.append(5 * u * (h.abs() @ w.abs().t() + b.abs()).view(len(tokens), hkv, d))
    angle = torch.tensor(positions).double()[:, None] * cfg.rope_theta ** (
        -torch.arange(0, d, 2).double() / d)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    k, e = plain[0], bound[0]
    if cfg.qk_norm:
        w = state[base + "self_attn.k_norm.weight"]
        size = (k.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt()
        least = size - e.norm(dim=-1, keepdim=True) / d ** 0.5
        assert least.min() > 0
        e = w * ((k.abs() + e) / least - k.abs() / size)
        k = k / size * w
    a, b = k.chunk(2, -1)
    both = (a.abs() + b.abs() + e[..., :d // 2] + e[..., d // 2:]).repeat(1, 1, 2)
    k = torch.cat((a * c - b * s, b * c + a * s), -1)
    e = (e[..., :d // 2] + e[..., d // 2:]).repeat(1, 1, 2)
    e = e + (32 * F + u if cfg.qk_norm else 3.1 * u + 400 * F) * both
    out = torch.stack((k, plain[1]), 1)
    error = torch.stack((e, bound[1]), 1)
    return out, error + (2.0 ** -22 if weights.dtype == torch.float16 else 0.0)


def rounded_logits(weights, tokens):
    """dense_logits with every result that the engine keeps in 16 bits rounded to them."""
    cfg, dtype = weights.config, weights.dtype
    state = {k: t.double() for k, t in weights.state_dict().items()}
    n, d = len(tokens), cfg.head_dim
    hq, hkv = cfg.num_attention_heads, cfg.num_key_value_heads

    def r(x):
        return x.to(dtype).double()

    def norm(x, w, inner=r):
        return r(inner(x / (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt()) * w)

    x = state["model.embed_tokens.weight"][torch.tensor(tokens)]
    angle = torch.arange(n).double()[:, None] * cfg.rope_theta ** (
        -torch.arange(0, d, 2).double() / d)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    causal = torch.full((n, n), -math.inf, dtype=torch.float64).triu(1)
    for i in range(cfg.num_hidden_layers):
        w = {k[len(f"model.layers.{i}."):]: t for k, t in state.items()
             if k.startswith(f"model.layers.{i}.")}
        h = norm(x, w["input_layernorm.weight"])
        q, k, v = (r(h @ w[f"self_attn.{m}_proj.weight"].t() + w[f"self_attn.{m}_proj.bias"])
                   for m in "qkv")
        heads = []
        for t, count, name in ((q, hq, "q"), (k, hkv, "k")):
            t = t.view(n, count, d)
            if cfg.qk_norm:
                y = t / (t.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt()
                a, b = (y * w[f"self_attn.{name}_norm.weight"]).chunk(2, -1)
                heads.append(r(torch.cat((a * c - b * s, b * c + a * s), -1)))
            else:
                a, b = t.chunk(2, -1)
                heads.append(r(torch.cat((r(a * r(c)) - r(b * r(s)),
                                          r(b * r(c)) + r(a * r(s))), -1)))
        q, k = heads[0], heads[1].repeat_interleave(hq // hkv, 1)
        v = v.view(n, hkv, d).repeat_interleave(hq // hkv, 1)
        scores = torch.einsum("thd,shd->hts", q, k) / math.sqrt(d) + causal
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        out = r(torch.einsum("hts,shd->thd", r(p), v) / p.sum(-1).t()[:, :, None])
        x = r(x + r(out.reshape(n, -1) @ w["self_attn.o_proj.weight"].t()))
        h = norm(x, w["post_attention_layernorm.weight"])
        gate, up = (r(h @ w[f"mlp.{m}_proj.weight"].t()) for m in ("gate", "up"))
        x = r(x + r(r(r(gate * torch.sigmoid(gate)) * up) @ w["mlp.down_proj.weight"].t()))
    return r(norm(x, state["model.norm.weight"]) @ state["lm_head.weight"].t())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_drafted_decoding_in_16_bits(dtype, qk_norm, monkeypatch):
    _, sequences = plain_run(qk_norm=qk_norm, dtype=dtype, page=4)
    engine = make_engine(qk_norm=qk_norm, dtype=dtype, page=4, logprobs=3,
                         drafter=Oracle(sequences, MODEL["vocab_size"]))
    add_requests(engine)
    watched, weights = Watched(engine, monkeypatch), engine.model
    checked = 0
    while engine.waiting or engine.running:
        layers = range(weights.config.num_hidden_layers)
        turns = {r.request_id: (r, len(r.generated)) for r in engine.running}
        history = {name: [watched.stored(name, i) for i in layers] for name in turns}
        watched.step()
        engine.cache.assert_invariants()
        names = list(turns)
        if not watched.layers:
            continue
        if watched.layers[0][0] != names:  # a prompt was admitted in this step
            assert watched.layers[0][0][:len(names)] == names
            (name,) = watched.layers[0][0][len(names):]
            request = engine.requests[name]
            turns[name] = (request, 1)
            if request.finished:  # nothing of it is stored any more
                continue
            # the prompt's rows: the store's, less what this step appended
            history[name] = [watched.stored(name, i)[:len(request.prompt)] for i in layers]
        check_attention(watched, history)
        checked += len(watched.layers)
        ids, q = watched.layers[0][:2]
        logits = watched.logits[-1].view(len(ids), q.shape[1], -1)
        for i, name in enumerate(ids):
            request, before = turns[name]
            tokens, nodes = walk(watched.trees[name], logits[i], None,
                                 request.max_new_tokens - before)
            assert request.generated[before:] == tokens
            check_scores(request.scores[before:], logits[i, nodes])
            if request.finished:
                continue
            for layer, (_, _, k, v, _) in enumerate(watched.layers):
                rows = watched.stored(name, layer)
                assert torch.equal(rows[:len(history[name][layer])], history[name][layer])
                added = torch.stack((k[i, nodes], v[i, nodes]), 1).cpu()
                assert torch.equal(rows[len(history[name][layer]):], added)
            sequence = request.prompt + request.generated[:-1]
            rows = watched.stored(name, 0).double()
            want, bound = first_layer_rows(weights, sequence, range(len(sequence)))
            assert ((rows - want).abs() <= bound).all()
            other, bound = first_layer_rows(weights, sequence, range(1, len(sequence) + 1))
            off = ((rows - other).abs() > bound).flatten(1).any(1)
            assert off.float().mean() > 0.5  # a position off by one would be seen
    assert engine.draft_stats["accepted"] > 20 and checked >= 9
    assert no_flags()

    # The whole forward: the engine's errors are sums of as many independent roundings as
    # rounded_logits makes (and of fp32 ones, far smaller), so of its size; the largest of
    # about a hundred rows of 320 differs between two such sums by well under a factor of 4.
    error = torch.zeros(3)
    dense = {}
    for name, r in engine.requests.items():
        tokens = r.prompt + r.generated
        exact, model = (t[len(r.prompt) - 1:-1] for t in
                        (dense_logits(weights, tokens), rounded_logits(weights, tokens)))
        logp, near = torch.log_softmax(exact, -1), torch.log_softmax(model, -1)
        entropy, near_entropy = (-(t.exp() * t).sum(-1) for t in (logp, near))
        dense[name] = exact, logp, entropy
        error = torch.maximum(error, torch.stack([
            (exact - model).abs().max(), (logp - near).abs().max(),
            (entropy - near_entropy).abs().max()]).float())
    of_logit, of_logp, of_entropy = (4 * error).tolist()
    for name, r in engine.requests.items():
        assert len(r.generated) == len(r.scores) == PROMPTS[name][1]
        for token, score, row, lp, h in zip(r.generated, r.scores, *dense[name]):
            assert abs(score.logprob - lp[token].item()) < of_logp
            assert abs(score.entropy - h.item()) < of_entropy
            assert row[token] > row.max() - 2 * of_logit
