"""BatchedEngine, DecodeBatch and RowCache over a cache held in 8 bits: the tokens of a
plain forward whose history goes through the tests' own 8-bit form."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from torch.nn import functional as F

import quantized_reference as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
MODEL = dict(vocab_size=256, hidden_size=128, intermediate_size=192, num_hidden_layers=2,
             num_attention_heads=4, num_key_value_heads=2)
PROMPTS = {"a": (37, 12), "b": (3, 14), "c": (16, 10)}


def make_engine(dtype=torch.float32, gpu_pages=300, page=8, union=256, seed=123, **options):
    from hisparse_b200.config import CacheConfig, HotConfig
    from hisparse_b200.engine import BatchedEngine, DecoderConfig, DecoderWeights, ServingCache

    weights = DecoderWeights.random(DecoderConfig(**MODEL), seed, device=DEV, dtype=dtype)
    cache = ServingCache(CacheConfig(gpu_pages=gpu_pages, host_pages=512, page_size=page,
                                     kv_heads=2, head_dim=32, device=DEV,
                                     dtype=torch.float8_e4m3fn), HotConfig(union, union))
    engine = BatchedEngine(weights, cache, **options)
    g = torch.Generator().manual_seed(21)
    for name, (length, new) in PROMPTS.items():
        engine.add_request(name, torch.randint(0, 256, (length,), generator=g).tolist(), new)
    return engine


def held(x):
    """The values that rows [N, heads, D] are held as, on the GPU in fp32."""
    return torch.from_numpy(ref.values(ref.records(x.double().cpu().numpy()), *x.shape[1:])).to(
        x.device, x.dtype)


def attend(q, k, v):
    """fp64 attention of q [Hq, D] over k, v [N, Hkv, D]."""
    group = q.shape[0] // k.shape[1]
    k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
    s = torch.einsum("hd,nhd->hn", q.double(), k) / math.sqrt(q.shape[1])
    return torch.einsum("hn,nhd->hd", torch.softmax(s, -1), v).to(q.dtype)


@torch.inference_mode()
def plain_tokens(weights, prompt, new):
    """Greedy tokens, their log probabilities, and the smallest gap between the two largest
    logits: the prompt over its exact rows, then every token over held rows, its own too."""
    n, layers = len(prompt), weights.config.num_hidden_layers
    x = F.embedding(torch.tensor(prompt, device=DEV), weights.embed)
    history = []
    for layer in range(layers):
        q, k, v = weights.project(layer, x, torch.arange(n, device=DEV).float())
        out = torch.stack([attend(q[i], k[:i + 1], v[:i + 1]) for i in range(n)])
        history.append((held(k), held(v)))
        x = weights.finish(layer, x, out)
    tokens, scores, gap = [], [], math.inf
    while True:
        logits = weights.logits(x[-1:])[0].double()
        top = logits.topk(2).values
        gap = min(gap, (top[0] - top[1]).item())
        tokens.append(int(logits.argmax()))
        scores.append(torch.log_softmax(logits, -1)[tokens[-1]].item())
        if len(tokens) == new:
            return tokens, scores, gap
        position = torch.tensor([n + len(tokens) - 1], device=DEV).float()
        x = F.embedding(torch.tensor(tokens[-1:], device=DEV), weights.embed)
        for layer in range(layers):
            q, k, v = weights.project(layer, x, position)
            k, v = (torch.cat(pair) for pair in zip(history[layer], (held(k), held(v))))
            history[layer] = (k, v)
            x = weights.finish(layer, x, attend(q[0], k, v)[None])


@pytest.fixture(scope="module")
def truth():
    """By request: tokens and log probabilities of the plain forward."""
    engine = make_engine()
    out = {}
    for name, (_, new) in PROMPTS.items():
        tokens, scores, gap = plain_tokens(engine.model, engine.requests[name].prompt, new)
        # Arithmetic in fp32 and another order changes logits by about 1e-5, and a K or V
        # element that lands on the other side of a border between codes by less than
        # 1e-2 in all; the seed was taken for its gap.
        assert gap > 2e-2, gap
        out[name] = (tokens, scores)
    return out


@pytest.mark.parametrize("gpu_pages", [300, 204])  # 204: the credits of three, no more
def test_engine_tokens(truth, gpu_pages):
    from hisparse_b200 import _lib

    engine = make_engine(gpu_pages=gpu_pages, logprobs=0)
    generated = engine.run()
    engine.cache.assert_invariants()
    assert generated == {name: tokens for name, (tokens, _) in truth.items()}
    for name, (_, scores) in truth.items():
        got = [s.logprob for s in engine.requests[name].scores]
        assert max(abs(a - b) for a, b in zip(got, scores)) < 1e-2
    misses = engine.cache.snapshot()["row_stats"]
    assert (misses["misses"] > 0) == (gpu_pages == 204)
    assert misses["h2d_bytes"] == misses["misses"] * 2 * 96
    assert not _lib.device_flags(DEV)


def test_engine_page_budget_of_everything(truth):
    """A Quest budget that covers the whole history selects all of it."""
    engine = make_engine(top_k=32)
    assert engine.run() == {name: tokens for name, (tokens, _) in truth.items()}


def test_engine_quest_budget_runs():
    """A budget below the history: tokens do not depend on where rows lie."""
    runs = [make_engine(top_k=3, gpu_pages=pages).run() for pages in (300, 204)]
    assert runs[0] == runs[1]


class Truth:
    """Drafts the true continuation beside a wrong branch."""

    def __init__(self, sequences):
        self.sequences = sequences

    def propose(self, tokens, limit):
        for sequence in self.sequences:
            if sequence[:len(tokens)] == tokens:
                out, parent = [], -1
                for token in sequence[len(tokens):len(tokens) + 4]:
                    out += [((token + 1) % 256, parent), (token, parent)]
                    parent = len(out) - 1
                return out[:limit]
        return []


@pytest.mark.parametrize("gpu_pages", [300, 204])
def test_engine_drafted_tokens(truth, gpu_pages):
    engine = make_engine(gpu_pages=gpu_pages)
    engine.drafter = Truth([engine.requests[name].prompt + tokens
                            for name, (tokens, _) in truth.items()])
    assert engine.run() == {name: tokens for name, (tokens, _) in truth.items()}
    assert engine.draft_stats["accepted"] > 15
    engine.cache.assert_invariants()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_engine_16_bit_models(dtype):
    """Placement changes nothing, drafted turns run, no flag is raised."""
    from hisparse_b200 import PromptLookup, _lib

    runs = [make_engine(dtype=dtype, gpu_pages=pages).run() for pages in (300, 204)]
    assert all(len(tokens) == PROMPTS[name][1] for name, tokens in runs[0].items())
    assert runs[0] == runs[1]
    drafted = make_engine(dtype=dtype, drafter=PromptLookup(), logprobs=2).run()
    assert {name: len(tokens) for name, tokens in drafted.items()} == \
        {name: new for name, (_, new) in PROMPTS.items()}
    assert not _lib.device_flags(DEV)


def test_metadata_bounds_the_held_rows():
    """Quest's bounds of every written page are those of the rows held in the host store."""
    engine = make_engine()
    for _ in range(6):
        engine.step()
    cache = engine.cache
    cache.rows.synchronize()
    host = cache.host.numpy()
    for res in cache.requests.values():
        for layer in range(res.layers):
            for page in range(-(-res.length // 8)):
                rows = min(8, res.length - 8 * page)
                keys = ref.values(host[res.host[layer, page], 0, :rows], 2, 32)
                low, high = (t[layer, page].double().cpu().numpy()
                             for t in (res.minimum, res.maximum))
                np.testing.assert_array_equal(low, keys.min(0))
                np.testing.assert_array_equal(high, keys.max(0))


def make_row_cache(b, length, p, hkv, d, hot_rows, seed):
    """A RowCache held in 8 bits with `b` requests of one layer, every other page resident."""
    from hisparse_b200 import CacheConfig, HotConfig, RowCache

    n = -(-length // p)
    hot = HotConfig(hot_rows // 2, hot_rows)
    config = CacheConfig(gpu_pages=b * (n + hot.hot_blocks(p)), host_pages=b * n, page_size=p,
                         kv_heads=hkv, head_dim=d, device=DEV, dtype=torch.float8_e4m3fn)
    x = np.random.default_rng(seed).standard_normal((b * n, 2, p, hkv, d))
    host = torch.from_numpy(ref.records(x))
    cache = RowCache(config, hot, host=host.pin_memory())
    cache.pool.zero_()
    minimum, maximum, block = {}, {}, 0
    for r in range(b):
        source, resident = np.arange(r * n, (r + 1) * n), np.full(n, -1)
        for page in list(range(0, n - 2, 2)) + [n - 2, n - 1]:
            resident[page] = block
            cache.pool[block] = host[source[page]].to(DEV)
            block += 1
        hot_blocks = list(range(block, block + hot.hot_blocks(p)))
        block += len(hot_blocks)
        cache.add_layer(r, 0, length, source, resident, hot_blocks)
        keys = ref.values(host.numpy()[source, 0], hkv, d)
        minimum[r], maximum[r] = (torch.from_numpy(t).to(torch.bfloat16)[None].to(DEV)
                                  for t in (keys.min(1), keys.max(1)))
    return cache, host, minimum, maximum


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_batch_layer_and_its_graph(dtype):
    """The batched hot path (selection, resolve, gather, both attention phases, merge) over
    the selected rows, eager and as a replayed graph."""
    from hisparse_b200 import DecodeBatch, _lib
    from hisparse_b200.batched import DecodeGraph

    b, length, p, hkv, d, hq, top = 2, 517, 16, 2, 64, 8, 9
    cache, host, minimum, maximum = make_row_cache(b, length, p, hkv, d, 2 * top * p, seed=3)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    batch = DecodeBatch(cache, range(b), 1, minimum, maximum, top, hq, streams=streams)

    def check(query, out):
        tokens, counts = batch.tokens.cpu().numpy(), batch.token_counts.cpu().tolist()
        for r in range(b):
            at = tokens[r, :counts[r]].astype(np.int64)
            rows = cache.tables[r, 0].source.cpu().numpy()[at // p].astype(np.int64) * p + at % p
            want, spread, size = ref.attend(query[r:r + 1].double().cpu().numpy(), host.numpy(),
                                            rows[None], hkv)
            bound = ref.attend_tolerance(want, spread, size, d, len(at), dtype)
            assert np.all(np.abs(out[r:r + 1].double().cpu().numpy() - want) <= bound)

    for step in range(3):
        query = torch.randn(b, hq, d, generator=torch.Generator().manual_seed(step)).to(DEV, dtype)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            out = batch.layer(0, query)
        torch.cuda.synchronize()
        check(query, out)
        assert batch.last_counts()[0, :, 2].min() >= 0
    assert batch.last_counts()[0, :, 1].sum() + batch.last_counts()[0, :, 2].sum() > 0
    graph = DecodeGraph([batch], 1, dtype=dtype)
    for step in range(3, 5):
        query = torch.randn(b, hq, d, generator=torch.Generator().manual_seed(step)).to(DEV, dtype)
        graph.queries[0][0].copy_(query)
        graph.replay()
        torch.cuda.synchronize()
        check(query, graph.outputs[0][0])
    assert not _lib.device_flags(DEV)


def test_row_cache_attention():
    """The reference's per-request entry point over a cache held in 8 bits."""
    from hisparse_b200 import Selection

    length, p, hkv, d, hq = 130, 8, 2, 32, 4
    cache, host, _, _ = make_row_cache(1, length, p, hkv, d, 256, seed=4)
    tokens = tuple(range(0, length, 2))
    selection = Selection.from_tokens(tokens, length, p, hq)
    query = torch.randn(hq, d, generator=torch.Generator().manual_seed(9)).to(DEV)
    for _ in range(2):  # the second time from the hot rows
        out = cache.attention(query, 0, 0, selection)
        want, spread, size = ref.attend(query[None].double().cpu().numpy(), host.numpy(),
                                        np.array([tokens]), hkv)
        bound = ref.attend_tolerance(want, spread, size, d, len(tokens), torch.float32)
        assert np.all(np.abs(out[None].double().cpu().numpy() - want) <= bound)
    assert cache.snapshot()["row_stats"]["hot_hits"] > 0


def test_engine_refusals():
    from hisparse_b200.batched import DecodeGraph  # noqa: F401
    from hisparse_b200.config import CacheConfig, HotConfig
    from hisparse_b200.engine import BatchedEngine, DecoderConfig, DecoderWeights, ServingCache

    weights = DecoderWeights.random(DecoderConfig(**MODEL), 5, device=DEV, dtype=torch.bfloat16)
    cache = ServingCache(CacheConfig(gpu_pages=100, kv_heads=2, head_dim=32, device=DEV),
                         HotConfig(64, 64))
    with pytest.raises(ValueError, match="dtype"):
        BatchedEngine(weights, cache)
