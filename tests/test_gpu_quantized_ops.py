"""The operators of a cache held in 8 bits against plain 64-bit forms: append_quantized,
read_quantized, attend_quantized."""

import math

import numpy as np
import pytest
import torch

import quantized_reference as ref
from hisparse_b200 import (CacheConfig, MappedHost, _lib, append_quantized, attend_quantized,
                           attend_rows, gather_rows, read_quantized)
from hisparse_b200.append import append_chunks, append_page
from hisparse_b200.row_index import RowPlan

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make_config(blocks, page, heads, dim):
    return CacheConfig(gpu_pages=blocks, page_size=page, kv_heads=heads, head_dim=dim, device=DEV,
                       dtype=torch.float8_e4m3fn)


def normal(*shape, seed=0, dtype=torch.float32, gain=None):
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(seed))
    if gain is not None:
        x = x * gain
    return x.to(dtype)


def make_pool(config, seed=0):
    """A pool of records of normal values with larger channels, as uint8 on the CPU."""
    rng = np.random.default_rng(seed)
    heads, dim = config.kv_heads, config.head_dim
    x = rng.standard_normal((config.gpu_pages, 2, config.page_size, heads, dim))
    x *= np.exp(0.7 * rng.standard_normal((heads, dim)))
    x *= np.exp(rng.standard_normal(x.shape[:4]))[..., None]  # rows of different sizes
    return ref.records(x)


class Pages:
    """Metadata of a call's chunks and its addresses."""

    def __init__(self, chunks, heads, dim, low=math.inf, high=-math.inf):
        shape = (chunks, heads, dim)
        self.minimum = torch.full(shape, low, dtype=torch.bfloat16, device=DEV)
        self.maximum = torch.full(shape, high, dtype=torch.bfloat16, device=DEV)
        self.summary = torch.full(shape, 7.0, device=DEV)

    def pointers(self):
        for t in (self.minimum, self.maximum, self.summary):
            yield t.data_ptr() + torch.arange(len(t), device=DEV) * t[0].numel() * t.element_size()


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def check_append(config, k, v, within, count, block, pool0, pages, pool, low0, high0):
    """Every byte of the pool, the bounds and the mean after an append to pool0."""
    heads, dim = config.kv_heads, config.head_dim
    expected = pool0.copy()
    for b, (w, n) in enumerate(zip(within, count)):
        for plane, x in enumerate((k, v)):
            expected[block[b], plane, w:w + n] = ref.records(x[b, :n].double().cpu().numpy())
    assert np.array_equal(pool.cpu().numpy(), expected)
    for b, (w, n) in enumerate(zip(within, count)):
        if n == 0:
            assert torch.all(pages.summary[b] == 7.0)
            continue
        held = ref.values(expected[block[b], 0, :w + n], heads, dim)
        new = held[w:]
        got = [t[b].double().cpu().numpy() for t in (pages.minimum, pages.maximum, pages.summary)]
        np.testing.assert_array_equal(got[0], np.minimum(low0, new.min(0)))
        np.testing.assert_array_equal(got[1], np.maximum(high0, new.max(0)))
        mean, size = held.mean(0), np.abs(held).sum(0) / (w + n)
        # w + n sums and one division in fp32, half a step each
        assert np.all((np.abs(got[2] - mean) <= (w + n + 1) * 2.0 ** -24 * size) |
                      (np.isnan(mean) & np.isnan(got[2])))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,page,within,count", [
    (2, 32, 16, [5, 0, 15], [1, 1, 1]),          # a decode step
    (8, 128, 16, [13, 0], [3, 16]),
    (4, 128, 64, [0, 0, 63], [64, 3, 1]),
    (1, 256, 12, [0, 11, 4], [12, 1, 0]),        # one chunk appends nothing
    (3, 80, 7, [2, 0], [5, 7]),
    (2, 33, 16, [3, 0], [9, 16]),                # no whole vectors
    (1, 1, 5, [0, 4], [5, 1]),
    (19, 16, 4, [1, 0], [3, 4]),                 # two groups of heads
    (16, 64, 130, [0, 65], [130, 65]),           # more rows than a tile keeps scales of
    (40, 24, 3, [0, 2], [3, 1]),
])
def test_append(dtype, heads, dim, page, within, count):
    chunks, tokens = len(within), max(max(count), 1)
    config = make_config(chunks + 2, page, heads, dim)
    pool0 = make_pool(config, seed=1)
    gain = torch.exp(normal(heads, dim, seed=2))
    k = normal(chunks, tokens, heads, dim, seed=3, dtype=dtype, gain=gain).to(DEV)
    v = normal(chunks, tokens, heads, dim, seed=4, dtype=dtype, gain=gain).to(DEV)
    block = [(i * 2 + 1) % (chunks + 2) for i in range(chunks)]
    pool = torch.from_numpy(pool0).to(DEV)
    pages = Pages(chunks, heads, dim, low=-0.5, high=0.25)
    append_quantized(k, v, ints(within), ints(count), ints(block, torch.int64), pool,
                     *pages.pointers(), config)
    check_append(config, k, v, within, count, block, pool0, pages, pool, -0.5, 0.25)
    assert not _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_special_values(dtype):
    """Zeros, numbers at the borders of a scale and of the type, subnormals, infinities,
    NaN: codes, scales and bounds; what is not finite is held as NaN."""
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    rows = [[0.0] * 8, [448.0] * 8, [449.0, 1, 1, 1, 0, 0, 0, 0], [top, -top, 1, 0, 0, 0, 0, 0],
            [tiny, -tiny / 2, 0, 0, 0, 0, 0, 0], [math.inf, 1.0, 2.0, -3.0, 0, 0, 0, 0],
            [math.nan] * 8, [-math.inf, math.nan, 0, -0.0, 1e-3, 2e-3, 0.875, -0.9375],
            [1.0625, 1.1875, 1.3125, -1.0625, 17.0, 19.0, 0.53125, 448.0],   # ties
            [448.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10, 2.0 ** -11, -2.0 ** -10, 0, 0]]
    k = torch.tensor(rows, dtype=torch.float64).to(dtype).view(1, len(rows), 1, 8).to(DEV)
    config = make_config(2, len(rows), 1, 8)
    pool0 = np.full((2, *config.page_shape), 9, dtype=np.uint8)
    pool = torch.from_numpy(pool0).to(DEV)
    pages = Pages(1, 1, 8)
    v = k.flip(1)
    append_quantized(k, v, ints([0]), ints([len(rows)]), ints([1], torch.int64), pool,
                     *pages.pointers(), config)
    expected = pool0.copy()
    for plane, x in enumerate((k, v)):
        expected[1, plane] = ref.records(x[0].double().cpu().numpy())
    assert np.array_equal(pool.cpu().numpy(), expected)
    held = torch.from_numpy(ref.values(expected[1, 0], 1, 8))
    for got, want in ((pages.minimum, held.amin(0)), (pages.maximum, held.amax(0))):
        assert torch.equal(got[0].double().cpu().nan_to_num(12345.0), want.nan_to_num(12345.0))


def test_append_in_pieces_equals_append_at_once():
    heads, dim, page = 4, 64, 16
    config = make_config(2, page, heads, dim)
    k, v = (normal(1, page, heads, dim, seed=s, dtype=torch.bfloat16).to(DEV) for s in (5, 6))
    pools, all_pages = [], []
    for cuts in ([0, 16], [0, 1, 2, 7, 16], list(range(17))):
        pool = torch.zeros((2, *config.page_shape), dtype=torch.uint8, device=DEV)
        pages = Pages(1, heads, dim)
        for a, b in zip(cuts, cuts[1:]):
            append_chunks(k[:, a:b], v[:, a:b], ints([a]), ints([b - a]), ints([1], torch.int64),
                          pool, *pages.pointers(), config)
        pools.append(pool)
        all_pages.append(pages)
    for pool, pages in zip(pools[1:], all_pages[1:]):
        assert torch.equal(pool, pools[0])
        assert torch.equal(pages.minimum, all_pages[0].minimum)
        assert torch.equal(pages.maximum, all_pages[0].maximum)
        # two sums of 16 numbers in another order: 16 half steps each
        held = read_quantized(pool, torch.arange(16, 32, device=DEV), config, torch.float32)[0]
        bound = 2 * 17 * 2.0 ** -24 * held.abs().mean(0)
        assert torch.all((pages.summary[0] - all_pages[0].summary[0]).abs() <= bound)


@pytest.mark.parametrize("heads,dim", [(2, 32), (3, 33), (8, 128)])
def test_append_host_mirror_and_host_only(heads, dim):
    page = 8
    config = make_config(3, page, heads, dim)
    host = torch.full((4, *config.page_shape), 3, dtype=torch.uint8).pin_memory()
    pool = torch.full((3, *config.page_shape), 5, dtype=torch.uint8, device=DEV)
    pages = Pages(3, heads, dim)
    k, v = (normal(3, 4, heads, dim, seed=s, dtype=torch.bfloat16).to(DEV) for s in (7, 8))
    within, count = [0, 4, 0], [4, 4, 2]
    append_quantized(k, v, ints(within), ints(count), ints([2, 0, -1], torch.int64), pool,
                     *pages.pointers(), config, MappedHost(host), ints([1, -1, 3], torch.int64))
    torch.cuda.synchronize()
    expected_pool = np.full(tuple(pool.shape), 5, dtype=np.uint8)
    expected_host = np.full(tuple(host.shape), 3, dtype=np.uint8)
    for b, (pb, hb) in enumerate(((2, 1), (0, None), (None, 3))):
        for plane, x in enumerate((k, v)):
            rec = ref.records(x[b, :count[b]].double().cpu().numpy())
            if pb is not None:
                expected_pool[pb, plane, within[b]:within[b] + count[b]] = rec
            if hb is not None:
                expected_host[hb, plane, within[b]:within[b] + count[b]] = rec
    assert np.array_equal(pool.cpu().numpy(), expected_pool)
    assert np.array_equal(host.numpy(), expected_host)
    # a second call on the host-only page reads its earlier rows there
    tail = Pages(1, heads, dim)
    append_quantized(k[:1], v[:1], ints([2]), ints([4]), ints([-1], torch.int64), pool,
                     *tail.pointers(), config, MappedHost(host), ints([3], torch.int64))
    torch.cuda.synchronize()
    held = ref.values(host.numpy()[3, 0, :6], heads, dim)
    size = np.abs(held).mean(0)
    assert np.all(np.abs(tail.summary[0].cpu().numpy() - held.mean(0)) <= 7 * 2.0 ** -24 * size)


def test_append_skips_bad_chunks():
    config = make_config(2, 8, 2, 32)
    pool = torch.full((2, *config.page_shape), 5, dtype=torch.uint8, device=DEV)
    pages = Pages(5, 2, 32)
    k = normal(5, 2, 2, 32).to(DEV)
    append_quantized(k, k, ints([0, 7, -1, 0, 1]), ints([2, 2, 1, 2, 2]),
                     ints([2, 0, 0, -1, 1], torch.int64), pool, *pages.pointers(), config)
    flags = _lib.device_flags(DEV)
    assert len(flags) == 1 and "beyond the pool" in flags[0]
    assert torch.all(pool[0] == 5) and torch.all(pool[1, :, 0] == 5) and not torch.all(pool[1] == 5)
    assert torch.all(pages.summary[:4] == 7.0) and not torch.any(pages.summary[4] == 7.0)


def test_append_views_and_page_form():
    heads, dim, page = 4, 32, 16
    config = make_config(2, page, heads, dim)
    fused = normal(3, 2, 3 * heads * dim, seed=9, dtype=torch.float16).to(DEV)
    k = fused[..., heads * dim:2 * heads * dim].unflatten(-1, (heads, dim))
    v = fused[..., 2 * heads * dim:].unflatten(-1, (heads, dim))
    pools = []
    for a, b in ((k, v), (k.contiguous(), v.contiguous()),
                 (k.transpose(2, 3).contiguous().transpose(2, 3), v)):
        pool = torch.zeros((2, *config.page_shape), dtype=torch.uint8, device=DEV)
        pages = Pages(1, heads, dim)
        append_quantized(a[:1], b[:1], ints([3]), ints([2]), ints([1], torch.int64), pool,
                         *pages.pointers(), config)
        pools.append(pool)
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])
    pool = torch.zeros((2, *config.page_shape), dtype=torch.uint8, device=DEV)
    append_page(pool, k[0], v[0], 1, 3, pages.minimum[0], pages.maximum[0], pages.summary[0],
                config)
    assert torch.equal(pool, pools[0])


def test_append_without_metadata_and_too_many_rows():
    config = make_config(3, 8, 2, 32)
    pool = torch.full((3, *config.page_shape), 5, dtype=torch.uint8, device=DEV)
    k = normal(3, 4, 2, 32, seed=14, dtype=torch.bfloat16).to(DEV)
    # the second chunk claims more rows than K has, the third a host block without a host
    append_quantized(k, k, ints([1, 0, 0]), ints([3, 5, 1]), ints([2, 1, 0], torch.int64), pool,
                     None, None, None, config, host_block=ints([-1, -1, 0], torch.int64))
    expected = np.full(tuple(pool.shape), 5, dtype=np.uint8)
    expected[2, :, 1:4] = ref.records(k[0, :3].double().cpu().numpy())
    assert np.array_equal(pool.cpu().numpy(), expected)
    assert "beyond the pool" in _lib.device_flags(DEV)[0]
    with pytest.raises(ValueError, match="go together"):
        at = ints([0, 0, 0], torch.int64)
        append_quantized(k, k, ints([0] * 3), ints([1] * 3), at, pool, at, None, at, config)


def test_append_nothing():
    config = make_config(2, 8, 2, 32)
    pool = torch.full((2, *config.page_shape), 5, dtype=torch.uint8, device=DEV)
    for shape in ((0, 3, 2, 32), (2, 0, 2, 32)):
        k = torch.zeros(shape, device=DEV)
        n = shape[0]
        append_quantized(k, k, ints([0] * n), ints([0] * n), ints([0] * n, torch.int64), pool,
                         None, None, None, config)
    assert torch.all(pool == 5) and not _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_strided_chunks(dtype):
    """Chunks a distance apart that vectors cannot step over, and expanded ones."""
    heads, dim = 2, 64
    config = make_config(4, 8, heads, dim)
    flat = normal(2000, seed=15, dtype=dtype).to(DEV)
    k = flat.as_strided((3, 2, heads, dim), (2 * heads * dim + 3, heads * dim, dim, 1))
    for source in (k, k[:1].expand(3, 2, heads, dim)):
        pool = torch.zeros((4, *config.page_shape), dtype=torch.uint8, device=DEV)
        append_quantized(source, source, ints([0, 2, 6]), ints([2, 2, 2]),
                         ints([3, 1, 0], torch.int64), pool, None, None, None, config)
        got = pool.cpu().numpy()
        for b, (block, w) in enumerate(((3, 0), (1, 2), (0, 6))):
            want = ref.records(source[b].double().cpu().numpy())
            for plane in range(2):
                assert np.array_equal(got[block, plane, w:w + 2], want)


# ---- reading back -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,page,count", [
    (2, 32, 16, 24), (8, 128, 16, 1), (4, 128, 64, 300), (1, 256, 12, 17), (3, 33, 5, 50),
    (2, 80, 16, 0), (1, 1, 3, 9), (19, 16, 4, 33)])
def test_read(dtype, heads, dim, page, count):
    config = make_config(9, page, heads, dim)
    pool = make_pool(config, seed=11)
    rows = np.random.default_rng(12).integers(0, 9 * page, count)
    rows[3::7] = -1
    got = read_quantized(torch.from_numpy(pool).to(DEV), torch.from_numpy(rows).to(DEV), config,
                         dtype)
    assert got.shape == (2, count, heads, dim) and got.dtype == dtype
    for plane in range(2):
        held = ref.values(ref.row_records(pool, np.maximum(rows, 0), plane), heads, dim)
        held[rows < 0] = 0.0
        # held values have 4 significant bits: exact but for fp16's range
        assert torch.equal(got[plane].cpu(), torch.from_numpy(held).float().to(dtype))


def test_read_shapes_bad_rows_and_nan():
    config = make_config(3, 4, 2, 16)
    pool = make_pool(config, seed=13)
    pool[1, 0, 2, 5] = 127
    rows = torch.tensor([[[6, 12], [-1, 2 ** 40]], [[11, 0], [-7, 6]]], device=DEV)
    got = read_quantized(torch.from_numpy(pool).to(DEV), rows, config)
    assert got.shape == (2, 2, 2, 2, 2, 16) and got.dtype == torch.bfloat16
    assert torch.isnan(got[0, 0, 0, 0, 0, 5]) and torch.isnan(got[0]).sum() == 2
    assert torch.all(got[:, 0, 0, 1] == 0) and torch.all(got[:, 0, 1] == 0)
    assert "beyond the pool" in _lib.device_flags(DEV)[0]
    strided = read_quantized(torch.from_numpy(pool).to(DEV), rows.flatten()[::2], config)
    assert torch.equal(strided[0, 0].nan_to_num(9.0), got[0, 0, 0, 0].nan_to_num(9.0))


@pytest.mark.parametrize("heads,dim,page", [(1, 33, 3), (2, 32, 16), (8, 128, 16), (16, 256, 5),
                                            (3, 80, 12)])
def test_gather_of_records(heads, dim, page):
    """Records begin anywhere in a line of 128 bytes, K's and V's not always at the same
    place; those that are not asked for stay as they are."""
    config = make_config(6, page, heads, dim)
    rng = np.random.default_rng(81)
    host = torch.from_numpy(rng.integers(0, 256, (9, *config.page_shape), dtype=np.uint8))
    pool0 = rng.integers(0, 256, (6, *config.page_shape), dtype=np.uint8)
    n = min(13, 2 * page)
    source, target = rng.permutation(9 * page)[:n], rng.permutation(6 * page)[:n]
    plan = [torch.from_numpy(np.append(x, [-1, -1])).to(DEV) for x in (source, target)]
    pool = torch.from_numpy(pool0).to(DEV)
    mapped = MappedHost(host.pin_memory())
    gather_rows(mapped, pool, RowPlan(None, *plan, None), config)
    for a, b in zip(source, target):
        pool0[b // page, :, b % page] = host[a // page, :, a % page]
    assert np.array_equal(pool.cpu().numpy(), pool0)


# ---- attention ----------------------------------------------------------------------------------
def check_attend(query, pool, rows, config, counts=None, run=None):
    heads, dim = config.kv_heads, config.head_dim
    got = (run or attend_quantized)(query.to(DEV), torch.from_numpy(pool).to(DEV),
                                    torch.from_numpy(rows).to(DEV), config,
                                    counts=None if counts is None else ints(counts))
    out, spread, size = ref.attend(query.double().numpy(), pool, rows, heads, counts)
    bound = ref.attend_tolerance(out, spread, size, dim, rows.shape[-1], query.dtype)
    assert got.dtype == query.dtype and got.shape == query.shape
    error = np.abs(got.double().cpu().numpy() - out)
    assert np.all(error <= bound), (np.nanmax(error / bound), np.isnan(error).sum())
    assert np.all(got.double().cpu().numpy()[out == 0] == 0) or out.any()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,q_heads,heads,dim,page,count", [
    (3, 8, 2, 32, 16, 160), (2, 32, 8, 128, 16, 300), (1, 28, 4, 128, 64, 700),
    (2, 16, 16, 64, 16, 129), (3, 10, 2, 80, 12, 77), (2, 12, 1, 256, 16, 200),
    (1, 4, 4, 128, 16, 1), (2, 2, 1, 33, 5, 40), (1, 1, 1, 1, 3, 9), (1, 40, 2, 64, 16, 90),
    (5, 6, 3, 96, 16, 257), (1, 18, 9, 192, 8, 65), (2, 9, 1, 128, 16, 1000),
    (1, 34, 17, 16, 16, 48), (1, 33, 1, 128, 16, 100), (1, 64, 2, 256, 16, 64)])
def test_attend(dtype, batch, q_heads, heads, dim, page, count):
    blocks = -(-batch * count // page) + 3
    config = make_config(blocks, page, heads, dim)
    pool = make_pool(config, seed=batch + dim)
    rng = np.random.default_rng(21)
    order = rng.permutation(blocks)[:, None] * page + np.arange(page)
    rows = order.reshape(-1)[:batch * count].reshape(batch, count).copy()
    loose = rows[:, count // 2:]
    loose[:] = rng.permuted(loose, axis=1)
    rows[:, 5::11] = -1
    query = normal(batch, q_heads, dim, seed=22, dtype=dtype)
    check_attend(query, pool, rows, config)
    counts = [max(0, count - 7 * i) for i in range(batch)]
    counts[-1] = 0 if batch > 1 else 1
    check_attend(query, pool, rows, config, counts)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,q_heads,heads,dim,count", [
    # 8, 4, 2 and 1 warps to a head; joined by a second kernel, in a cluster, or not at all
    (2, 7, 1, 128, 1000), (1, 12, 1, 256, 2000), (1, 5, 1, 64, 100), (160, 12, 1, 256, 100),
    (3, 14, 2, 128, 400), (60, 6, 2, 96, 900), (80, 24, 2, 256, 300),
    (2, 28, 4, 128, 300), (53, 28, 4, 128, 700), (1, 28, 4, 128, 2500), (160, 4, 4, 64, 250),
    (2, 16, 8, 64, 500), (1, 32, 16, 80, 3000), (150, 8, 8, 32, 260)])
def test_attend_joins(dtype, batch, q_heads, heads, dim, count):
    """Requests share a pool; one of them has a few rows only, so that most of the parts
    that are joined saw nothing."""
    config = make_config(70, 16, heads, dim)
    pool = make_pool(config, seed=dim + heads)
    rows = np.random.default_rng(41).integers(0, 70 * 16, (batch, count))
    rows[0, 3:] = -1
    query = normal(batch, q_heads, dim, seed=42, dtype=dtype)
    some = sorted({0, batch // 3, batch - 1})  # compared
    for counts in (None, [count - i % 45 for i in range(batch - 1)] + [33]):
        got = attend_quantized(query.to(DEV), torch.from_numpy(pool).to(DEV),
                               torch.from_numpy(rows).to(DEV), config,
                               counts=None if counts is None else ints(counts))
        check_attend(query[some], pool, rows[some], config,
                     None if counts is None else [counts[i] for i in some],
                     run=lambda *_, **__: got[some])


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_nothing_to_see(dtype):
    config = make_config(4, 16, 2, 64)
    pool = make_pool(config, seed=31)
    query = normal(3, 8, 64, dtype=dtype)
    rows = np.full((3, 50), -1)
    rows[1, 49] = 7
    got = check_attend(query, pool, rows, config)
    assert torch.all(got[0] == 0) and torch.all(got[2] == 0) and torch.all(got[1].abs().amax(-1) > 0)
    got = check_attend(query, pool, np.zeros((3, 0), dtype=np.int64), config)
    assert torch.all(got == 0)
    check_attend(query, pool, np.abs(rows), config, [-3, 99, 0])
    assert not _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_bad_rows_are_skipped(dtype):
    config = make_config(4, 16, 2, 128)
    pool = make_pool(config, seed=32)
    rows = np.random.default_rng(33).integers(0, 64, (2, 90))
    rows[0, 3:40:2] = 64
    rows[1, 80] = 2 ** 45
    check_attend(normal(2, 4, 128, dtype=dtype), pool, rows, config)
    assert "beyond the pool" in _lib.device_flags(DEV)[0]


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_unseen_rows_take_no_part(dtype):
    """NaN codes in rows that are masked or behind the counts."""
    config = make_config(8, 16, 2, 128)
    pool = make_pool(config, seed=34)
    clean = pool.copy()
    pool[4:] = 127
    rows = np.concatenate([np.arange(64), 64 + np.arange(64)])[None].repeat(2, 0)
    query = normal(2, 8, 128, seed=35, dtype=dtype)
    got = check_attend(query, pool, rows, config, [64, 37])
    assert torch.isfinite(got).all()
    assert torch.equal(got, check_attend(query, clean, rows, config, [64, 37]))
    rows[:, 64:] = -1
    rows[1, 37:] = -1
    check_attend(query, pool, rows, config)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [128, 33])
def test_attend_rows_never_written(dtype, dim):
    """Records of zeros are not seen, wherever they are in the list."""
    config = make_config(8, 16, 2, dim)
    pool = make_pool(config, seed=62)
    pool[2], pool[5, :, 3:] = 0, 0
    rows = np.random.default_rng(63).permutation(128)[None].repeat(2, 0)
    query = normal(2, 8, dim, seed=64, dtype=dtype)
    written = pool[rows // 16, 0, rows % 16].any(-1)
    got = check_attend(query, pool, np.where(written, rows, -1), config)
    same = attend_quantized(query.to(DEV), torch.from_numpy(pool).to(DEV),
                            torch.from_numpy(rows).to(DEV), config)
    assert torch.equal(same, got)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_nan_is_kept(dtype):
    """A NaN in a seen K makes its heads NaN, one in a seen V its element."""
    config = make_config(4, 16, 2, 128)
    pool = make_pool(config, seed=36)
    pool[1, 1, 3, 128 + 9] = 255          # V of row 19, KV head 1, element 9
    query = normal(1, 4, 128, seed=37, dtype=dtype).to(DEV)
    rows = torch.arange(40, device=DEV)[None]
    got = attend_quantized(query, torch.from_numpy(pool).to(DEV), rows, config)
    assert torch.isnan(got[0, 2:, 9]).all() and torch.isnan(got).sum() == 2
    pool[1, 0, 3, 5] = 127                # K of row 19, KV head 0
    got = attend_quantized(query, torch.from_numpy(pool).to(DEV), rows, config)
    assert torch.isnan(got[0, :2]).all() and torch.isnan(got).sum() == 2 * 128 + 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low,high", [(-100, -100), (100, 100), (-90, 90), (-20, 0)])
def test_attend_scales_far_apart(dtype, low, high):
    """V rows whose sizes differ by many powers of two, and K rows with tiny ones."""
    if dtype == torch.float16 and high > 0:
        pytest.skip("results leave fp16's range")
    config = make_config(8, 16, 1, 64)
    pool = make_pool(config, seed=38)
    pool[:, 1, :, 64] = np.random.default_rng(39).integers(low, high + 1, (8, 16)) + 127
    pool[::2, 0, :, 64] = 27
    check_attend(normal(1, 4, 64, seed=40, dtype=dtype), pool, np.arange(128)[None], config)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gain", [30.0, 1e-3])
def test_attend_sharp_and_flat(dtype, gain):
    """Scores of hundreds (one row takes all, the maximum moves) and of almost nothing."""
    config = make_config(20, 16, 2, 128)
    pool = make_pool(config, seed=41)
    check_attend(normal(1, 8, 128, seed=42, dtype=dtype) * gain, pool, np.arange(320)[None], config)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_rows_of_each_head(dtype):
    config = make_config(8, 16, 2, 64)
    pool = make_pool(config, seed=43)
    rows = np.random.default_rng(44).integers(-1, 128, (2, 6, 70))
    query = normal(2, 6, 64, seed=45, dtype=dtype)
    check_attend(query, pool, rows, config)
    device = torch.from_numpy(pool).to(DEV)
    shared = torch.from_numpy(rows[:, :1]).to(DEV)
    expected = attend_quantized(query.to(DEV), device, shared[:, 0], config)
    assert torch.equal(attend_quantized(query.to(DEV), device, shared.expand(2, 6, 70), config),
                       expected)
    for i in range(2):  # the form of one request
        one = attend_rows(query[i].to(DEV), device, shared[i, 0], config)
        assert (one - expected[i]).abs().max() <= 2.0 ** -6 * expected[i].abs().max()
        assert torch.equal(one, attend_rows(query[i].to(DEV), device,
                                            shared[i].expand(6, 70), config))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_strides(dtype):
    """Queries inside a fused projection, rows as a view, rows of an odd distance."""
    config = make_config(8, 16, 2, 64)
    pool = make_pool(config, seed=46)
    device = torch.from_numpy(pool).to(DEV)
    fused = normal(3, 8 * 64 + 7, seed=47, dtype=dtype).to(DEV)
    rows = torch.from_numpy(np.random.default_rng(48).integers(-1, 128, (3, 90))).to(DEV)
    for view, at in ((fused[:, :512].unflatten(-1, (8, 64)), rows),
                     (fused[:, 5:517].unflatten(-1, (8, 64)), rows),
                     (fused[:, :512].unflatten(-1, (64, 8)).transpose(1, 2), rows),
                     (fused[:, :512].unflatten(-1, (8, 64)), rows[:, 1:78]),
                     (fused[:, :512].unflatten(-1, (8, 64)), rows[:, ::2])):
        got = attend_quantized(view, device, at, config)
        plain = attend_quantized(view.contiguous().clone(), device, at.contiguous().clone(), config)
        bound = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -9
        assert (got - plain).abs().max() <= bound * plain.abs().max()


def test_attend_far_rows():
    """Rows whose byte offsets pass 32 bits."""
    heads, dim, page = 8, 128, 16
    blocks = (1 << 32) // (2 * page * 1056) + 40
    config = make_config(blocks, page, heads, dim)
    pool = torch.zeros((blocks, *config.page_shape), dtype=torch.uint8, device=DEV)
    small = make_config(4, page, heads, dim)
    data = make_pool(small, seed=49)
    pool[-4:] = torch.from_numpy(data).to(DEV)
    rows = torch.arange(64, device=DEV)[None]
    query = normal(1, 32, dim, seed=50, dtype=torch.bfloat16).to(DEV)
    near = attend_quantized(query, torch.from_numpy(data).to(DEV), rows, small)
    far = attend_quantized(query, pool, rows + (blocks - 4) * page, config)
    assert torch.equal(near, far)
    held = read_quantized(pool, rows[0] + (blocks - 4) * page, config)
    assert torch.equal(held, read_quantized(torch.from_numpy(data).to(DEV), rows[0], small))
    pages = Pages(1, heads, dim)
    k = normal(1, 1, heads, dim, seed=51, dtype=torch.bfloat16).to(DEV)
    append_quantized(k, k, ints([15]), ints([1]), ints([blocks - 1], torch.int64), pool,
                     *pages.pointers(), config)
    assert np.array_equal(pool[-1, 0, 15].cpu().numpy(),
                          ref.records(k[0, 0].double().cpu().numpy()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,group", [(8, 4), (4, 7), (17, 2), (1, 12), (3, 5)])
def test_attend_many_units(dtype, heads, group):
    """Enough rows that every warp goes around its rings of rows and of scales several
    times, on one split and on many, with runs, single rows and masked ones."""
    batch, count, dim, page = 40, 1200, 64, 16
    blocks = 200
    config = make_config(blocks, page, heads, dim)
    pool = make_pool(config, seed=65)
    rng = np.random.default_rng(66)
    rows = rng.integers(0, blocks * page, (batch, count))
    runs = rng.integers(0, blocks, (batch, count // 32))
    for i in range(0, count // 32 - 1, 2):  # every other unit two runs
        rows[:, 32 * i:32 * i + 16] = runs[:, i:i + 1] * page + np.arange(16)
        rows[:, 32 * i + 16:32 * i + 32] = runs[:, i + 1:i + 2] * page + np.arange(16)
    rows[:, 7::29] = -1
    query = normal(batch, heads * group, dim, seed=67, dtype=dtype)
    device = torch.from_numpy(pool).to(DEV)
    got = attend_quantized(query.to(DEV), device, torch.from_numpy(rows).to(DEV), config)
    for b in (0, 17, 39):
        out, spread, size = ref.attend(query[b:b + 1].double().numpy(), pool, rows[b:b + 1], heads)
        bound = ref.attend_tolerance(out, spread, size, dim, count, dtype)
        assert np.all(np.abs(got[b:b + 1].double().cpu().numpy() - out) <= bound)
        alone = attend_quantized(query[b:b + 1].to(DEV), device,
                                 torch.from_numpy(rows[b:b + 1]).to(DEV), config)
        assert np.all(np.abs(alone.double().cpu().numpy() - out) <= bound)
    assert not _lib.device_flags(DEV)


# ---- streams, graphs, refusals --------------------------------------------------------------------
def test_append_read_attend_together_in_a_graph():
    """A step as it is used (append a row, attend, read the rows), captured and replayed with
    new inputs, equals the same calls outside of a graph."""
    heads, dim, page, batch = 4, 128, 16, 3
    config = make_config(12, page, heads, dim)
    pool0 = torch.from_numpy(make_pool(config, seed=61)).to(DEV)
    rows = torch.arange(3 * 64, device=DEV).view(3, 64)
    k, v = (torch.zeros(batch, 1, heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    query = torch.zeros(batch, 16, dim, dtype=torch.bfloat16, device=DEV)
    within, count = ints([15, 3, 0]), ints([1, 1, 1])
    block = ints([3, 5, 9], torch.int64)

    def step(pool, pages, pointers):
        append_quantized(k, v, within, count, block, pool, *pointers, config)
        return (attend_quantized(query, pool, rows, config),
                read_quantized(pool, rows, config))

    pool, pages = pool0.clone(), Pages(batch, heads, dim)
    pointers = list(pages.pointers())
    step(pool, pages, pointers)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(pool, pages, pointers)
    for seed in (1, 2):
        for i, t in enumerate((k, v, query)):
            t.copy_(normal(*t.shape, seed=10 * seed + i, dtype=torch.bfloat16))
        pool.copy_(pool0)
        graph.replay()
        other, more = pool0.clone(), Pages(batch, heads, dim)
        eager = step(other, more, list(more.pointers()))
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)
        assert torch.equal(pool, other)


def test_two_streams():
    """Calls that overlap on two streams have workspaces of their own."""
    config = make_config(64, 16, 4, 128)
    pool = torch.from_numpy(make_pool(config, seed=71)).to(DEV)
    rows = torch.stack([torch.randperm(1024, generator=torch.Generator().manual_seed(s))
                        for s in range(2)]).to(DEV)
    queries = [normal(1, 28, 128, seed=s, dtype=torch.bfloat16).to(DEV) for s in range(2)]
    expected = [attend_quantized(q, pool, rows[i:i + 1], config) for i, q in enumerate(queries)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(attend_quantized(queries[i], pool, rows[i:i + 1], config))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, expected[i]) for r in results[i])


def test_refusals():
    config = make_config(4, 16, 2, 64)
    pool = torch.zeros((4, *config.page_shape), dtype=torch.uint8, device=DEV)
    query = torch.zeros(1, 4, 64, device=DEV)
    rows = torch.zeros((1, 8), dtype=torch.int64, device=DEV)
    plain = CacheConfig(gpu_pages=4, kv_heads=2, head_dim=64, device=DEV)

    def refuse(match, call, *args, **kwargs):
        with pytest.raises(ValueError, match=match):
            call(*args, **kwargs)

    refuse("8 bits", attend_quantized, query, pool, rows, plain)
    refuse("pool must be", attend_quantized, query, pool[..., :-1], rows, config)
    refuse("pool must be", read_quantized, pool.view(torch.int8), rows, config)
    refuse("query must be", attend_quantized, query[0], pool, rows, config)
    refuse("query must be", attend_quantized, query[..., :32], pool, rows, config)
    refuse("GQA", attend_quantized, query[:, :3], pool, rows, config)
    refuse("element type", attend_quantized, query.double(), pool, rows, config)
    refuse("rows must be", attend_quantized, query, pool, rows.int(), config)
    refuse("rows must be", attend_quantized, query, pool, rows[0], config)
    refuse("rows must be", attend_quantized, query, pool, rows.expand(2, 8), config)
    refuse("counts must be", attend_quantized, query, pool, rows, config, rows[0, :1])
    refuse("no backward", attend_quantized, query.requires_grad_(), pool, rows, config)
    refuse("element type", read_quantized, pool, rows, config, torch.float64)
    refuse("rows must be", read_quantized, pool, rows.int(), config)
    k = torch.zeros(1, 2, 2, 64, device=DEV)
    one, at = ints([1]), rows[0, :1]

    def append(k=k, v=k, within=one, block=at, minimum=at, host=None, config=config, pool=pool):
        append_quantized(k, v, within, one, block, pool, minimum, at, at, config, host)

    refuse("matching", append, v=k[:, :1])
    refuse("matching", append, k=k[0], v=k[0])
    refuse("must both", append, v=k.half())
    refuse("must both", append, k=k.double(), v=k.double())
    refuse("within must be", append, within=at)
    refuse("pool_block must be", append, block=one)
    refuse("minimum_ptrs must be", append, minimum=rows[0, :2])
    refuse("8 bits", append, config=plain)
    host = torch.zeros((4, 2, 16, 2, 64)).pin_memory()
    refuse("layouts differ", append, host=MappedHost(host))
