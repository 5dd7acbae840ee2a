"""BatchedEngine's drafted decoding, log probabilities and head norms against the
engine's own plain decoding and a dense fp64 forward of the same weights."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
MODEL = dict(vocab_size=320, hidden_size=128, intermediate_size=192, num_hidden_layers=3,
             num_attention_heads=4, num_key_value_heads=2)


def make_engine(qk_norm=False, dtype=torch.float32, seed=3, gpu_pages=400, page=16, union=512,
                **options):
    from hisparse_b200.config import CacheConfig, HotConfig
    from hisparse_b200.engine import BatchedEngine, DecoderConfig, DecoderWeights, ServingCache

    config = DecoderConfig(**MODEL, qk_norm=qk_norm)
    weights = DecoderWeights.random(config, seed, device=DEV, dtype=dtype)
    cache = ServingCache(CacheConfig(gpu_pages=gpu_pages, host_pages=1024, page_size=page,
                                     kv_heads=2, head_dim=32, device=DEV, dtype=dtype),
                         HotConfig(union, union))
    return BatchedEngine(weights, cache, **options)


PROMPTS = {"a": (41, 25), "b": (3, 31), "c": (64, 14), "d": (17, 1), "e": (90, 30)}


def add_requests(engine, repeat=True, names="abcde"):
    g = torch.Generator().manual_seed(11)
    for name, (length, new) in PROMPTS.items():
        piece = torch.randint(0, MODEL["vocab_size"], (13,), generator=g).tolist()
        prompt = (piece * 8)[:length] if repeat else \
            torch.randint(0, MODEL["vocab_size"], (length,), generator=g).tolist()
        if name in names:
            engine.add_request(name, prompt, new)


class Oracle:
    """Proposes the true continuation (from a plain run) beside wrong branches."""

    def __init__(self, truth, vocab, depth=5, wrong=2, stop_after=None):
        self.truth, self.vocab = truth, vocab
        self.depth, self.wrong, self.stop_after = depth, wrong, stop_after

    def propose(self, tokens, limit):
        for sequence in self.truth:
            if sequence[:len(tokens)] == tokens:
                out, parent = [], -1
                for d, token in enumerate(sequence[len(tokens):len(tokens) + self.depth]):
                    for i in range(self.wrong):
                        out.append(((token + 1 + i) % self.vocab, parent))
                    if self.stop_after is not None and d >= self.stop_after:
                        token = (token + 100) % self.vocab  # the path goes wrong here
                    out.append((token, parent))
                    parent = len(out) - 1
                return out[:limit]
        return []


def plain_run(**options):
    engine = make_engine(**options)
    add_requests(engine)
    out = engine.run()
    return out, [r.prompt + r.generated for r in engine.requests.values()]


def no_flags():
    from hisparse_b200 import _lib

    return not _lib.device_flags(DEV)


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("drafter", ["lookup", "oracle", "stops", "wrong", "deep", "empty"])
def test_drafted_decoding_emits_the_plain_tokens(qk_norm, drafter):
    """fp32: the greedy tokens do not depend on how they are drafted (the smallest
    top-2 margin of the plain run is far above fp32's differences, checked here).
    Small pages, so that accepted paths cross one and two page borders."""
    from hisparse_b200 import PromptLookup

    want, sequences = plain_run(qk_norm=qk_norm, page=4)
    v = MODEL["vocab_size"]
    drafters = {"lookup": PromptLookup(depth=6, branches=3), "oracle": Oracle(sequences, v),
                "stops": Oracle(sequences, v, stop_after=2), "wrong": Oracle(sequences, v, 1, 3, 0),
                "deep": Oracle(sequences, v, depth=12, wrong=4), "empty": Oracle([], v)}
    engine = make_engine(qk_norm=qk_norm, page=4, drafter=drafters[drafter], logprobs=2)
    add_requests(engine)
    steps = 0
    while engine.waiting or engine.running:
        engine.step()
        steps += 1
        engine.cache.assert_invariants()
    assert {n: r.generated for n, r in engine.requests.items()} == want
    for r in engine.requests.values():
        assert len(r.scores) == len(r.generated)
        assert all(s.top[0][0] == t and s.top[0][1] == s.logprob
                   for s, t in zip(r.scores, r.generated))
        assert min(s.top[0][1] - s.top[1][1] for s in r.scores) > 1e-4
    stats = engine.draft_stats
    if drafter in ("oracle", "deep"):
        assert stats["accepted"] >= 60 and steps < 25
    if drafter == "wrong":
        assert stats["accepted"] == 0 and stats["drafted"] > 0
    if drafter == "empty":
        assert stats == {"steps": 0, "drafted": 0, "accepted": 0}
    assert not engine.cache.requests and len(engine.cache.free_pool) == 400
    assert no_flags()


def test_drafted_decoding_through_the_gather_and_eos():
    """A pool with one request's credits keeps no history resident: the tree reads
    gathered rows. An end token inside an accepted path ends the request there."""
    want, sequences = plain_run()
    eos = want["a"][9]
    plain, _ = plain_run(eos_token_id=eos)
    engine = make_engine(gpu_pages=110, drafter=Oracle(sequences, MODEL["vocab_size"]),
                         eos_token_id=eos)
    add_requests(engine)
    assert engine.run() == plain
    assert engine.cache.snapshot()["row_stats"]["misses"] > 0
    assert engine.draft_stats["accepted"] > 0 and no_flags()


def test_drafted_decoding_with_cancellation_bf16():
    from hisparse_b200 import PromptLookup

    engine = make_engine(qk_norm=True, dtype=torch.bfloat16, drafter=PromptLookup(), logprobs=0)
    add_requests(engine)
    for _ in range(4):
        engine.step()
    engine.cancel("b")
    engine.cache.assert_invariants()
    out = engine.run()
    assert all(len(out[n]) == PROMPTS[n][1] for n in "acde")
    assert all(len(r.scores) == len(r.generated) and all(s.top == () for s in r.scores)
               for r in engine.requests.values())
    assert no_flags()


def dense_logits(weights, tokens):
    """fp64 logits of every position of a token list: the formulas, layer by layer."""
    cfg = weights.config
    state = {k: v.double() for k, v in weights.state_dict().items()}
    n, d = len(tokens), cfg.head_dim
    hq, hkv = cfg.num_attention_heads, cfg.num_key_value_heads

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + cfg.rms_norm_eps).sqrt() * w

    x = state["model.embed_tokens.weight"][torch.tensor(tokens)]
    angle = torch.arange(n).double()[:, None] * cfg.rope_theta ** (
        -torch.arange(0, d, 2).double() / d)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    causal = torch.full((n, n), -math.inf, dtype=torch.float64).triu(1)
    for i in range(cfg.num_hidden_layers):
        base = f"model.layers.{i}."
        w = {k[len(base):]: v for k, v in state.items() if k.startswith(base)}
        h = norm(x, w["input_layernorm.weight"])
        q, k, v = (h @ w[f"self_attn.{m}_proj.weight"].t() + w[f"self_attn.{m}_proj.bias"]
                   for m in "qkv")
        heads = []
        for t, count, name in ((q, hq, "q"), (k, hkv, "k")):
            t = t.view(n, count, d)
            if cfg.qk_norm:
                t = norm(t, w[f"self_attn.{name}_norm.weight"])
            a, b = t.chunk(2, -1)
            heads.append(torch.cat((a * c - b * s, b * c + a * s), -1))
        q, k = heads[0], heads[1].repeat_interleave(hq // hkv, 1)
        v = v.view(n, hkv, d).repeat_interleave(hq // hkv, 1)
        p = torch.softmax(torch.einsum("thd,shd->hts", q, k) / math.sqrt(d) + causal, -1)
        x = x + torch.einsum("hts,shd->thd", p, v).reshape(n, -1) @ w["self_attn.o_proj.weight"].t()
        h = norm(x, w["post_attention_layernorm.weight"])
        gate, up = h @ w["mlp.gate_proj.weight"].t(), h @ w["mlp.up_proj.weight"].t()
        x = x + (gate * torch.sigmoid(gate) * up) @ w["mlp.down_proj.weight"].t()
    return norm(x, state["model.norm.weight"]) @ state["lm_head.weight"].t()


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("drafted", [False, True])
def test_scores_equal_a_dense_forward(qk_norm, drafted):
    """Every emitted token is the dense forward's argmax and its log probability,
    entropy and alternatives are that forward's. Three layers of fp32 (products
    of at most 192 terms) keep logits of size ~1 to 1e-4; bound 2e-3."""
    from hisparse_b200 import PromptLookup

    engine = make_engine(qk_norm=qk_norm, logprobs=5, drafter=PromptLookup() if drafted else None)
    add_requests(engine, names="abc")
    engine.run()
    for r in engine.requests.values():
        logits = dense_logits(engine.model, r.prompt + r.generated)[len(r.prompt) - 1:-1]
        logp = torch.log_softmax(logits, -1)
        assert logits.argmax(-1).tolist() == r.generated
        for row, token, score in zip(logp, r.generated, r.scores):
            assert abs(score.logprob - row[token].item()) < 2e-3
            assert abs(score.entropy + (row.exp() * row).sum().item()) < 2e-3
            assert len(score.top) == 5
            for other, value in score.top:
                assert abs(value - row[other].item()) < 2e-3
            assert score.top[4][1] > row.topk(5).values[4].item() - 2e-3


def test_scores_do_not_change_the_tokens():
    want, _ = plain_run()
    engine = make_engine(logprobs=32)
    add_requests(engine)
    assert engine.run() == want
    engine = make_engine(top_k=2, dtype=torch.bfloat16)
    add_requests(engine)
    sparse = engine.run()
    engine = make_engine(top_k=2, dtype=torch.bfloat16, logprobs=3)
    add_requests(engine)
    assert engine.run() == sparse


def test_refusals():
    with pytest.raises(ValueError, match="logprobs"):
        make_engine(logprobs=33)
    with pytest.raises(ValueError, match="logprobs"):
        make_engine(logprobs=-1)
    with pytest.raises(ValueError, match="top_k must be None"):
        make_engine(top_k=2, drafter=Oracle([], 1))
    engine = make_engine(drafter=Oracle([], 1))
    add_requests(engine, names="a")
    engine.step()
    with pytest.raises(ValueError, match="leaves its page"):
        engine.cache.plan_append(["a"], [17])
    with pytest.raises(ValueError, match="leaves its page"):
        engine.cache.plan_append(["a"], [0])
