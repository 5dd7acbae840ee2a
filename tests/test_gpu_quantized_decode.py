"""DecodeBatch over a cache held in 8 bits: the two phases in every query type, requests whose KV
heads are split over shards, and what is refused."""

import numpy as np
import pytest
import torch

import quantized_bounds as bounds
import quantized_reference as ref
from hisparse_b200 import (CacheConfig, DecodeBatch, HotConfig, MappedHost, RowCache, _lib,
                           gather_rows)
from hisparse_b200.batched import DecodeGraph
from hisparse_b200.row_index import RowPlan
from hisparse_b200.sharded import head_slice

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
BATCH, LENGTH, PAGE, TOP = 2, 517, 16, 9


def cache_of(x):
    """A RowCache of rows x [BATCH, pages, 2, PAGE, Hkv, D], every other page resident, with the
    metadata of its requests and its host store."""
    b, n, _, p, heads, dim = x.shape
    hot = HotConfig(TOP * p, 2 * TOP * p)
    config = CacheConfig(gpu_pages=b * (n + hot.hot_blocks(p)), host_pages=b * n, page_size=p,
                         kv_heads=heads, head_dim=dim, device=DEV, dtype=torch.float8_e4m3fn)
    host = torch.from_numpy(ref.records(x.reshape(b * n, 2, p, heads, dim)))
    cache = RowCache(config, hot, host=host.pin_memory())
    cache.pool.zero_()
    low, high, block = {}, {}, 0
    for r in range(b):
        source, resident = np.arange(r * n, (r + 1) * n), np.full(n, -1)
        for page in list(range(0, n - 2, 2)) + [n - 2, n - 1]:
            resident[page] = block
            cache.pool[block] = host[source[page]].to(DEV)
            block += 1
        hot_blocks = list(range(block, block + hot.hot_blocks(p)))
        block += len(hot_blocks)
        cache.add_layer(r, 0, LENGTH, source, resident, hot_blocks)
        keys = ref.values(host.numpy()[source, 0], heads, dim)
        low[r], high[r] = (torch.from_numpy(t).to(torch.bfloat16)[None].to(DEV)
                           for t in (keys.min(1), keys.max(1)))
    return cache, low, high, host.numpy()


def rows_of(heads, dim, seed):
    x = np.random.default_rng(seed).standard_normal(
        (BATCH, -(-LENGTH // PAGE), 2, PAGE, heads, dim))
    x[:, :, 0] *= 0.5
    return x


def queries(q_heads, dim, dtype, seed):
    return torch.randn(BATCH, q_heads, dim, generator=torch.Generator().manual_seed(seed)).to(
        DEV, dtype)


def check(batch, cache, host, query, out):
    heads = cache.config.kv_heads
    tokens, counts = batch.tokens.cpu().numpy(), batch.token_counts.cpu().tolist()
    for r in range(BATCH):
        at = tokens[r, :counts[r]].astype(np.int64)
        rows = cache.tables[r, 0].source.cpu().numpy()[at // PAGE].astype(np.int64) * PAGE + at % PAGE
        want, bound = bounds.attend(query[r:r + 1].double().cpu().numpy(), host, rows[None], heads,
                                    query.dtype)
        assert np.all(np.abs(out[r:r + 1].double().cpu().numpy() - want) <= bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_heads,heads,dim", [(8, 2, 64), (28, 4, 128), (6, 2, 33)])
def test_two_phases(dtype, q_heads, heads, dim):
    """Eager, into a given result, and as a replayed graph."""
    cache, low, high, host = cache_of(rows_of(heads, dim, seed=dim))
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    batch = DecodeBatch(cache, range(BATCH), 1, low, high, TOP, q_heads, streams=streams)
    out = torch.empty(BATCH, q_heads, dim, dtype=dtype, device=DEV)
    for step in range(2):
        query = queries(q_heads, dim, dtype, step)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            got = batch.layer(0, query, out)
        torch.cuda.synchronize()
        assert got is out
        check(batch, cache, host, query, out)
    assert batch.last_counts()[0, :, 2].sum() > 0  # rows that were gathered
    graph = DecodeGraph([batch], 1, dtype=dtype)
    query = queries(q_heads, dim, dtype, 2)
    graph.queries[0][0].copy_(query)
    graph.replay()
    torch.cuda.synchronize()
    check(batch, cache, host, query, graph.outputs[0][0])
    assert not _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", TYPES)
def test_kv_heads_split_over_shards(monkeypatch, dtype):
    """The shards' batches run one after another here, with the exchange between them; they
    select what one batch of all heads does and attend over their own heads."""
    import torch.distributed as dist

    from hisparse_b200 import sharded

    q_heads, heads, dim, shards = 8, 4, 64, 2
    x = rows_of(heads, dim, seed=91)
    whole, low, high, host = cache_of(x)
    plain = DecodeBatch(whole, range(BATCH), 1, low, high, TOP, q_heads)
    query = queries(q_heads, dim, dtype, 92)
    expected = plain.layer(0, query)
    check(plain, whole, host, query, expected)
    monkeypatch.setattr(dist, "get_world_size", lambda *_: shards)
    monkeypatch.setattr(sharded, "same_on_every_rank", lambda *_: True)
    parts = []
    for rank in range(shards):
        ks, qs = head_slice(heads, q_heads, rank, shards)
        cache, low, high, host = cache_of(x[:, :, :, :, ks])
        batch = DecodeBatch(cache, range(BATCH), 1, low, high, TOP, q_heads // shards,
                            group="both", streams=(torch.cuda.Stream(), torch.cuda.Stream()))
        parts.append((batch, cache, host, query[:, qs].contiguous(), qs))
    torch.cuda.synchronize()

    def run(part, batch, own):
        with torch.cuda.stream(batch.compute):
            out = batch.layer(0, own, part=part)
        torch.cuda.synchronize()
        return out

    for batch, *_, own, _ in parts:
        run("head", batch, own)
    partials = torch.stack([batch.partial for batch, *_ in parts])

    def exchange(batch):
        batch.partials.copy_(partials)

    monkeypatch.setattr(DecodeBatch, "exchange", exchange)
    for batch, cache, host, own, qs in parts:
        batch.exchange()
        out = run("tail", batch, own)
        assert torch.equal(batch.tokens, plain.tokens)
        check(batch, cache, host, own, out)
        graph = DecodeGraph([batch], 1, dtype=dtype)  # in two pieces around the exchange
        assert graph.segmented
        graph.queries[0][0].copy_(own)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(batch.tokens, plain.tokens)
        check(batch, cache, host, own, graph.outputs[0][0])
    assert not _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 33])
def test_merge_of_one_phase(dtype, dim):
    """A merge joins as many phases as it is told; what the other one left is not looked at."""
    batch, q_heads, heads, count = 3, 8, 2, 300
    pool = bounds.pool_of(25, PAGE, heads, dim, seed=dim)
    rows = np.stack([np.random.default_rng(s).permutation(400)[:count] for s in range(batch)])
    query = torch.randn(batch, q_heads, dim, generator=torch.Generator().manual_seed(5)).to(DEV, dtype)
    lib, code, stream = _lib.load(), _lib.dtype_code(dtype), _lib.stream_of(DEV)
    nbytes = lib.hs_attend_quantized_workspace_bytes(batch, 2, code, q_heads, heads, dim, count)
    workspace = torch.full((nbytes,), 255, dtype=torch.uint8, device=DEV)  # NaN
    device, at = torch.from_numpy(pool).to(DEV), torch.from_numpy(rows).to(DEV)
    given = torch.tensor([[300, 7], [150, 7], [0, 7]], device=DEV)
    out = torch.empty_like(query)
    _lib.check(lib.hs_attend_quantized_phase(
        batch, query.data_ptr(), q_heads * dim, code, device.data_ptr(), 25, at.data_ptr(), count,
        count, given.data_ptr(), 2, 0, 1, 0, q_heads, heads, dim, PAGE, workspace.data_ptr(), nbytes,
        None, stream))
    _lib.check(lib.hs_attend_quantized_merge(batch, 1, out.data_ptr(), code, q_heads, heads, dim,
                                             count, workspace.data_ptr(), nbytes, stream))
    want, bound = bounds.attend(query.double().cpu().numpy(), pool, rows, heads, dtype,
                                [300, 150, 0])
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound)
    assert torch.all(out[2] == 0)


def test_graph_of_a_plain_cache_takes_its_dtype():
    hot = HotConfig(TOP * PAGE, TOP * PAGE)
    config = CacheConfig(gpu_pages=40, host_pages=8, page_size=PAGE, kv_heads=2, head_dim=32,
                         device=DEV, dtype=torch.bfloat16)
    cache = RowCache(config, hot)
    cache.add_layer(0, 0, 20, [0, 1], [0, 1], list(range(2, 2 + hot.hot_blocks(PAGE))))
    low = {0: torch.zeros(1, 2, 2, 32, dtype=torch.bfloat16, device=DEV)}
    batch = DecodeBatch(cache, [0], 1, low, low, TOP, 4,
                        streams=(torch.cuda.Stream(), torch.cuda.Stream()))
    with pytest.raises(ValueError, match="the cache's dtype"):
        DecodeGraph([batch], 1, dtype=torch.float32)
    assert DecodeGraph([batch], 1, dtype=torch.bfloat16).outputs[0].dtype == torch.bfloat16


def test_gather_refuses_other_records():
    """Pool and host store agree with each other but not with the configuration."""
    def store(dim, page):
        config = CacheConfig(gpu_pages=2, page_size=page, kv_heads=2, head_dim=dim, device=DEV,
                             dtype=torch.float8_e4m3fn)
        return config, torch.zeros((2, *config.page_shape), dtype=torch.uint8)

    config, own = store(64, 8)
    row = torch.zeros(1, dtype=torch.int64, device=DEV)
    plan = RowPlan(None, row, row, None)
    others = [store(32, 8)[1], store(64, 4)[1], torch.zeros(2, 2, 8, 2, 64, dtype=torch.float16)]
    for other in others:
        with pytest.raises(ValueError, match="pool must be"):
            gather_rows(MappedHost(other.pin_memory()), other.to(DEV), plan, config)
    gather_rows(MappedHost(own.pin_memory()), own.to(DEV), plan, config)
