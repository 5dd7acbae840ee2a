"""attend_quantized within bounds that one missing row, or a weight in fewer bits, exceeds."""

import numpy as np
import pytest
import torch

import quantized_bounds as bounds
import quantized_reference as ref
from hisparse_b200 import CacheConfig, _lib, attend_quantized

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]

# batch, query heads, KV heads, head_dim, rows: 8, 4, 2 and 1 warps to a head, one to four quads
# of query heads, splits joined by a second kernel, in a cluster, or none
FLAT = [(1, 28, 4, 128, 1200), (60, 28, 4, 128, 700), (3, 32, 8, 128, 300), (2, 16, 1, 128, 1000),
        (2, 14, 1, 64, 1200), (150, 10, 2, 80, 260), (2, 12, 1, 256, 600), (1, 32, 16, 64, 900),
        (2, 8, 8, 32, 500), (2, 6, 2, 33, 400)]
CANCELLING = [(1, 28, 4, 128, 40), (1, 16, 2, 64, 64), (1, 16, 1, 128, 33), (1, 12, 1, 256, 50),
              (1, 8, 2, 32, 24), (1, 32, 8, 128, 40)]


def normal(*shape, seed, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def flat(batch, q_heads, heads, dim, count, dtype):
    """Scores of about 0.3: weights from a half to twice their mean."""
    pool = bounds.pool_of(-(-count // 16) + 2, 16, heads, dim, seed=count + dim)
    rng = np.random.default_rng(dim)
    rows = np.stack([rng.permutation(len(pool) * 16)[:count] for _ in range(batch)])
    return normal(batch, q_heads, dim, seed=1, dtype=dtype), pool, rows


def cancelling(batch, q_heads, heads, dim, count, dtype):
    """Scores of two products; results of one query head of each KV head nearly cancel."""
    pool = bounds.pool_of(-(-count // 16) + 1, 16, heads, dim, seed=7 + count, key_size=1.5,
                          key_elements=2)
    query = normal(batch, q_heads, dim, seed=dim, dtype=dtype) * dim ** 0.5 / 4
    rows = np.random.default_rng(count).permutation(len(pool) * 16)[:count]
    some = bounds.cancel(query[0].double().numpy(), pool, rows, heads, q_heads // heads - 1)
    return query, pool, rows[None], some


def run(query, pool, rows, heads, counts=None):
    config = CacheConfig(gpu_pages=len(pool), page_size=pool.shape[2], kv_heads=heads,
                         head_dim=query.shape[-1], device=DEV, dtype=torch.float8_e4m3fn)
    got = attend_quantized(query.to(DEV), torch.from_numpy(pool).to(DEV),
                           torch.from_numpy(rows).to(DEV), config, counts)
    assert got.dtype == query.dtype and not _lib.device_flags(DEV)
    return got.double().cpu().numpy()


def check(got, query, pool, rows, heads, dtype):
    out, bound = bounds.attend(query.double().numpy(), pool, rows, heads, dtype)
    error = np.abs(got - out)
    assert np.all(error <= bound), (error / bound).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", FLAT)
def test_every_row_counts(dtype, case):
    query, pool, rows = flat(*case, dtype)
    got = run(query, pool, rows, case[2])
    some = sorted({0, case[0] // 2, case[0] - 1})
    check(got[some], query[some], pool, rows[some], case[2], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CANCELLING)
def test_small_differences(dtype, case):
    query, pool, rows, some = cancelling(*case, dtype)
    got = run(query, pool, rows, case[2])
    check(got, query, pool, rows, case[2], dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_heads,heads,dim", [(8, 2, 64), (28, 4, 128), (12, 1, 256), (6, 2, 33)])
def test_nothing_seen_whatever_the_query(dtype, q_heads, heads, dim):
    """Zeros where no row is seen (masked, beyond the pool, never written, behind the counts),
    also for queries that are not finite; those are NaN where a row is seen."""
    pool = bounds.pool_of(4, 16, heads, dim, seed=5)
    pool[3] = 0
    rows = np.stack([np.full(70, -1), np.arange(70) % 16 + 48, np.full(70, 64), np.arange(70) % 48,
                     np.arange(70) % 48, np.full(70, -1)])
    rows[4, 1:] = -1
    query = normal(6, q_heads, dim, seed=6, dtype=dtype)
    query[:5, 0, 0], query[:5, -1, -1], query[:5, 1] = np.inf, np.nan, -np.inf
    config = CacheConfig(gpu_pages=4, page_size=16, kv_heads=heads, head_dim=dim, device=DEV,
                         dtype=torch.float8_e4m3fn)
    counts = torch.tensor([70, 70, 70, 0, 70, 70], dtype=torch.int32, device=DEV)
    some = [0, 1, q_heads - 1]  # the heads that are not finite
    for limit in (counts, None):
        got = attend_quantized(query.to(DEV), torch.from_numpy(pool).to(DEV),
                               torch.from_numpy(rows).to(DEV), config, limit)
        assert torch.all(got[[0, 1, 2, 5]] == 0)
        seen = got[4:5] if limit is not None else got[3:5]
        assert torch.isnan(seen[:, some]).all()
        others = [h for h in range(q_heads) if h not in some]
        assert torch.isfinite(seen[:, others]).all()
        if limit is not None:
            assert torch.all(got[3] == 0)
    assert "beyond the pool" in _lib.device_flags(DEV)[0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_heads,heads,dim", [(8, 2, 64), (8, 2, 128), (28, 4, 128), (4, 1, 256),
                                               (6, 2, 33)])
def test_tail_behind_one_row(dtype, q_heads, heads, dim):
    """Rows of one small weight behind a row that takes nearly all, which has no part in half of
    the elements. The weights, 2^-24 of the largest, differ from head to head."""
    rng = np.random.default_rng(dim)
    x = np.zeros((3, 2, 16, heads, dim))
    x[0, 0, 3, :, 0] = 1.0
    x[:, 1] = 256 * rng.standard_normal((3, 16, heads, dim))
    x[0, 1, 3, :, dim // 2:] = 0
    pool, rows = ref.records(x), np.arange(32)[None]
    query = torch.zeros(1, q_heads, dim)
    query[0, :, 0] = (24 + torch.arange(q_heads) / q_heads) * np.log(2) * dim ** 0.5
    query = query.to(dtype)
    check(run(query, pool, rows, heads), query, pool, rows, heads, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,q_heads,heads,dim,count", [
    (4, 32, 8, 128, 1000), (1, 8, 2, 64, 3000), (3, 16, 16, 80, 400), (2, 6, 6, 32, 250),
    (60, 4, 2, 96, 100), (1, 12, 1, 256, 300), (2, 5, 1, 48, 33), (1, 18, 2, 16, 8000)])
def test_joins_of_the_cuda_core_kernel(dtype, batch, q_heads, heads, dim, count):
    """Rows of each head, and queries off their vectors' boundary with shared rows: splits in a
    cluster, with a workspace, or none; few rows, so that some splits see nothing, and none."""
    pool = bounds.pool_of(40, 16, heads, dim, seed=count + dim)
    rng = np.random.default_rng(count)
    rows = rng.integers(0, 640, (batch, q_heads, count))
    rows[0, 0, 20:] = -1
    rows[-1, -1] = -1
    query = normal(batch, q_heads, dim, seed=2, dtype=dtype)
    some = sorted({0, batch - 1})
    got = run(query, pool, rows, heads)
    check(got[some], query[some], pool, rows[some], heads, dtype)
    assert np.all(got[-1, -1] == 0)
    counts = torch.full((batch,), count // 2, dtype=torch.int32, device=DEV)
    got = run(query, pool, rows, heads, counts)
    check(got[some], query[some], pool, rows[some][..., :count // 2], heads, dtype)
    shared = rows[:, 0]
    device = torch.zeros(batch * q_heads * dim + 1, dtype=dtype, device=DEV)
    aside = device[1:].view(batch, q_heads, dim)  # an element past the boundary
    aside.copy_(query)
    config = CacheConfig(gpu_pages=len(pool), page_size=16, kv_heads=heads, head_dim=dim,
                         device=DEV, dtype=torch.float8_e4m3fn)
    got = attend_quantized(aside, torch.from_numpy(pool).to(DEV),
                           torch.from_numpy(shared).to(DEV), config).double().cpu().numpy()
    check(got[some], query[some], pool, shared[some], heads, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_heads,dim", [(8, 16), (64, 16), (8, 128), (8, 256), (8, 24)])
def test_millions_of_rows_of_zeros(dtype, q_heads, dim):
    """V rows of zeros have the smallest scale, which makes their terms of the sum the largest
    numbers, more so when scores rise by less than what moves the maximum; the last rows of the
    request hold something."""
    count, heads = 1 << 21, 8
    x = np.zeros((1, 2, 3, heads, dim))
    x[0, 0, 0, :, 0], x[0, 0, 1:, :, 0] = -1.0, 1.0
    x[0, 1, 2] = 256 * np.random.default_rng(dim).standard_normal((heads, dim))
    pool = ref.records(x)
    query = torch.zeros(1, q_heads, dim)
    query[..., 0] = 3.75 * np.log(2) * dim ** 0.5  # weights of 2^3.75 and 2^-3.75
    query = query.to(dtype)
    # row 0 in the first unit of every part that the request may be split into, row 2 at its end
    rows = torch.where(torch.arange(count, device=DEV) // 32 % 512 == 0, 0, 1)[None]
    rows[0, -32:] = 2
    config = CacheConfig(gpu_pages=1, page_size=3, kv_heads=heads, head_dim=dim, device=DEV,
                         dtype=torch.float8_e4m3fn)
    got = attend_quantized(query.to(DEV), torch.from_numpy(pool).to(DEV), rows, config)
    k, v = (ref.values(pool[0, plane], heads, dim) for plane in range(2))
    w = np.exp(k[:, 0] @ query[0, 0].double().numpy() / np.sqrt(dim))
    w *= [128 * 32, count - 129 * 32, 32]
    want = np.repeat(w[2] / w.sum() * v[2], q_heads // heads, 0)
    # a sum of 2^21 terms in fp32, a step each at most; every other error is far below
    bound = 2.0 ** -2 * np.abs(want) + torch.finfo(dtype).smallest_normal
    assert np.all(np.abs(got[0].double().cpu().numpy() - want) <= bound)


def test_a_million_rows_of_zeros_on_cuda_cores():
    """So many requests that each would have one split, whose sums fp32 could not hold."""
    count, batch, dim = (1 << 20) + 64, 296, 9
    x = np.zeros((1, 2, 2, 1, dim))
    x[0, 1, 1] = np.arange(1, dim + 1)
    pool = ref.records(x)
    query = torch.ones(batch, 1, dim)
    rows = torch.zeros(count, dtype=torch.int64, device=DEV)
    rows[-16:] = 1
    config = CacheConfig(gpu_pages=1, page_size=2, kv_heads=1, head_dim=dim, device=DEV,
                         dtype=torch.float8_e4m3fn)
    got = attend_quantized(query.to(DEV), torch.from_numpy(pool).to(DEV), rows.expand(batch, count),
                           config).double().cpu().numpy()
    want = 16 / count * x[0, 1, 1, 0]
    # sums of 2^20 equal terms, a step of fp32 each at most
    assert np.all(np.abs(got - want) <= 2.0 ** -3 * want)


def test_cluster_of_the_cuda_core_kernel_in_a_graph():
    """Captured with rows of each head and replayed with others."""
    pool = bounds.pool_of(20, 16, 2, 64, seed=3)
    config = CacheConfig(gpu_pages=20, page_size=16, kv_heads=2, head_dim=64, device=DEV,
                         dtype=torch.float8_e4m3fn)
    device = torch.from_numpy(pool).to(DEV)
    query = normal(2, 8, 64, seed=4, dtype=torch.bfloat16).to(DEV)
    rows = torch.zeros(2, 8, 200, dtype=torch.int64, device=DEV)
    attend_quantized(query, device, rows, config)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = attend_quantized(query, device, rows, config)
    for seed in range(3):
        rows.copy_(torch.from_numpy(np.random.default_rng(seed).integers(-1, 320, rows.shape)))
        graph.replay()
        check(captured.double().cpu().numpy(), query.cpu(), pool, rows.cpu().numpy(), 2,
              torch.bfloat16)
