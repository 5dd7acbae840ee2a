"""A drafted step over a cache held in 8 bits attends to the values held, as plain steps do."""

import math

import numpy as np
import pytest
import torch

import quantized_reference as ref
from hisparse_b200 import CacheConfig, DecodeBatch, HotConfig, RowCache, _lib, tree_mask
from test_gpu_verify_ops import F, assert_within, half_step, tree_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
LENGTHS, PAGE, Q_HEADS, HEADS, DIM, NODES, TOP = (101, 64), 8, 8, 2, 64, (5, 3), 13


def rows_like(generator, *shape):
    """Rows with elements at the top of fp16 where queries are small, and a KV head whose
    values are small."""
    x = torch.randn(*shape, HEADS, DIM, generator=generator)
    x[..., 1, :] *= 2.0 ** -6
    x[..., 7] = torch.tensor([65504.0, -64000.0]).repeat(math.prod(shape))[:x[..., 7].numel()].view(
        x[..., 7].shape)
    return x


def flip(x):
    """Every other row's large elements with the other sign."""
    x[..., ::2, :, 7] *= -1
    return x


def make_cache(generator, dtype, change=lambda x: x):
    """Every page in the host store, the first and the last two of a request resident."""
    n = -(-max(LENGTHS) // PAGE)
    hot = HotConfig(TOP * PAGE, TOP * PAGE)
    b = len(LENGTHS)
    config = CacheConfig(gpu_pages=b * (n + hot.hot_blocks(PAGE)), host_pages=b * n, page_size=PAGE,
                         kv_heads=HEADS, head_dim=DIM, device=DEV, dtype=torch.float8_e4m3fn)
    rows = rows_like(generator, b * n, 2, PAGE).to(dtype)
    rows[:, 1] = change(rows[:, 1])
    host = torch.from_numpy(ref.records(rows.double().numpy()))
    cache = RowCache(config, hot, host=host.pin_memory())
    cache.pool.zero_()
    block, bounds = 0, {}
    for r, length in enumerate(LENGTHS):
        pages = -(-length // PAGE)
        source, resident = np.arange(r * n, r * n + pages), np.full(pages, -1)
        for page in {0, pages - 2, pages - 1}:
            resident[page], block = block, block + 1
            cache.pool[resident[page]] = host[source[page]].to(DEV)
        hot_blocks = list(range(block, block + hot.hot_blocks(PAGE)))
        block += len(hot_blocks)
        cache.add_layer(r, 0, length, source, resident, hot_blocks)
        bounds[r] = torch.zeros((1, n, HEADS, DIM), dtype=torch.bfloat16, device=DEV)
    return cache, host, bounds, n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("signs", [False, True])
def test_layer_tree_over_held_values(dtype, signs):
    """With large V elements of one sign, results of 65,536 (infinity in fp16) among them, and
    of both."""
    g = torch.Generator().manual_seed(17)
    change = flip if signs else lambda x: x
    cache, host, bounds, n = make_cache(g, dtype, change)
    batch = DecodeBatch(cache, range(len(LENGTHS)), 1, bounds, bounds, TOP, Q_HEADS)
    b, t = len(LENGTHS), max(NODES)
    query = torch.randn(b, t, Q_HEADS, DIM, generator=g)
    query[..., 7] = 2.0 ** -14
    query = query.to(DEV, dtype)
    key, value = (rows_like(g, b, t).to(DEV, dtype) for _ in range(2))
    value = change(value)
    mask = tree_mask([[-1, 0, 0, 1, 3], [-1, 0, 1]], DEV)
    counts = torch.tensor(LENGTHS, dtype=torch.int32, device=DEV)
    nodes = torch.tensor(NODES, dtype=torch.int32, device=DEV)
    positions = torch.full((b, TOP * PAGE), -1, dtype=torch.int32)
    for r, length in enumerate(LENGTHS):
        positions[r, :length] = torch.arange(length)
    out = batch.layer_tree(0, query, key, value, mask, nodes, positions.to(DEV), counts)
    # the definition over the values held, history and nodes
    held = [torch.from_numpy(ref.values(ref.records(x.double().cpu().numpy()), HEADS, DIM))
            for x in (key, value)]
    pool = torch.from_numpy(ref.values(host.numpy(), HEADS, DIM))
    rows = torch.where(positions >= 0, positions + torch.arange(b)[:, None] * n * PAGE, -1).long()
    want, size, _ = tree_reference(query, *held, mask, pool, rows, counts, nodes)
    u, keys = half_step(dtype), rows.shape[1] + t
    # The bound of attend_tree, with the sum of a score's products in place of the norms,
    # which the large elements meet only small ones in; weights of fp16 queries are not rounded
    # below fp32.
    reach = max(
        torch.einsum("thgd,nhd->thgn", query[r].double().cpu().abs().unflatten(1, (HEADS, -1)),
                     torch.cat((held[0][r], pool[rows[r, :LENGTHS[r]] // PAGE, 0,
                                                 rows[r, :LENGTHS[r]] % PAGE])).abs()).max()
        for r in range(b)).item() / math.sqrt(DIM)
    relative = 2 * (DIM + 4) * F * reach + (keys + 32) * F + (u if dtype == torch.bfloat16 else 0)
    bound = relative * size + u * (want.abs() + relative * size)
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
        # 65,520 and more rounds to infinity; all results of these are above, or far below
        large = want.abs() > 65520
        assert torch.all((want.abs() - 65520).abs() > relative * size) and large.any() != signs
        want = torch.where(large, torch.sign(want) * math.inf, want)
    assert out.dtype == dtype
    assert_within(out, want, bound)
    assert not _lib.device_flags(DEV)


def test_layer_tree_takes_one_dtype():
    g = torch.Generator().manual_seed(18)
    cache, _, bounds, _ = make_cache(g, torch.float16)
    batch = DecodeBatch(cache, range(2), 1, bounds, bounds, TOP, Q_HEADS)
    query = torch.zeros(2, 1, Q_HEADS, DIM, dtype=torch.float16, device=DEV)
    key = torch.zeros(2, 1, HEADS, DIM, device=DEV)
    mask = torch.ones((2, 1), dtype=torch.int64, device=DEV)
    one = torch.ones(2, dtype=torch.int32, device=DEV)
    positions = torch.zeros((2, TOP * PAGE), dtype=torch.int32, device=DEV)
    for k, v in ((key, key), (key.half(), key), (key, key.half())):
        with pytest.raises(ValueError, match="one dtype"):
            batch.layer_tree(0, query, k, v, mask, one, positions, one)


def test_held_values_in_another_type():
    from hisparse_b200.quantized import held_values

    config = CacheConfig(kv_heads=HEADS, head_dim=DIM, device=DEV, dtype=torch.float8_e4m3fn)
    k = rows_like(torch.Generator().manual_seed(19), 2, 3).half()
    want = torch.from_numpy(ref.values(ref.records(k.double().numpy()), HEADS, DIM))
    for dtype in (torch.float32, torch.bfloat16):
        got = held_values(k.to(DEV), k.to(DEV), config, dtype)
        assert got.dtype == dtype and got.shape == (2, *k.shape)
        assert torch.equal(got[0].double().cpu(), want) and torch.equal(got[0], got[1])
    assert held_values(k.to(DEV), k.to(DEV), config).dtype == torch.float16
