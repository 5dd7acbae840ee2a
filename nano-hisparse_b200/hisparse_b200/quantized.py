"""A cache held in 8 bits: rows quantised as they are written
(``append_quantized``), read back (``read_quantized``) and attended to by decode
queries (``attend_quantized``).

Every miss of the resolver crosses the host link and every selected row crosses
HBM, so the bytes of a row are what a decode step costs; here they are halved
against 16 bits. One token's K (or V) is a record of e4m3 codes, a power-of-two
scale for each KV head, and padding to a multiple of 32 bytes: the scale belongs
to the row because ``resolve_rows`` and ``gather_rows`` move rows alone. The
formulas stand in include/hisparse_quantized.h.

``CacheConfig(dtype=torch.float8_e4m3fn)`` selects such a cache; ``append_chunks``,
``append_page``, ``attend_rows``, ``row_attention``, ``RowCache``, ``DecodeBatch`` and
``BatchedEngine`` then take these operators by themselves.
"""

from __future__ import annotations

from dataclasses import replace

import torch

from . import _lib

_VALUES = (torch.float32, torch.float16, torch.bfloat16)


def check_pool(pool, config):
    """Blocks of a pool held in 8 bits; raises if it is not one of `config`."""
    if not config.quantized:
        raise ValueError("config must hold its rows in 8 bits (dtype torch.float8_e4m3fn)")
    shape = pool.shape
    if pool.dtype != torch.uint8 or shape[1:] != config.page_shape or not pool.is_contiguous():
        raise ValueError("pool must be contiguous uint8 [blocks, 2, page_size, row_bytes]")
    return shape[0]


def append_quantized(k, v, within, count, pool_block, pool, minimum_ptrs, maximum_ptrs,
                     summary_ptrs, config, host=None, host_block=None):
    """Quantise and append one page chunk per batch item b: ``append_chunks`` for a
    pool held in 8 bits.

    k, v: [B, T, Hkv, D] of one of the three value dtypes (chunk b uses rows
    0..count[b]-1); within, count: int32 [B]; pool_block: int64 [B];
    minimum_ptrs / maximum_ptrs / summary_ptrs: int64 [B] device pointers to the
    page's [Hkv, D] bounds (bfloat16) and fp32 mean, both of the values held
    (all three None: no metadata);
    host: MappedHost of the pinned store (uint8, of the pool's page shape) and
    host_block int64 [B] (-1: no mirror; pool_block -1: host only). Chunks of one
    call must touch distinct pages. Runs on the current stream.
    """
    index = _lib.one_device(k, v, within, count, pool_block, pool, minimum_ptrs, maximum_ptrs,
                            summary_ptrs, host_block)
    blocks = check_pool(pool, config)
    shape = k.shape
    if v.shape != shape or len(shape) != 4 or shape[2:] != (config.kv_heads, config.head_dim):
        raise ValueError("expected matching [batch, tokens, kv_heads, head_dim] K/V")
    if k.dtype not in _VALUES or v.dtype != k.dtype:
        raise ValueError("K and V must both be float32, float16 or bfloat16")
    if host is not None and (host.tensor.dtype != torch.uint8
                             or host.tensor.shape[1:] != config.page_shape
                             or not host.tensor.is_contiguous()):
        raise ValueError("host store and pool layouts differ")
    batch, tokens = shape[:2]
    if (minimum_ptrs is None) != (maximum_ptrs is None) or \
            (minimum_ptrs is None) != (summary_ptrs is None):
        raise ValueError("bounds and mean go together: all three addresses or none")
    limits = []  # addresses
    for name, t, dt in (("within", within, torch.int32), ("count", count, torch.int32),
                        ("pool_block", pool_block, torch.int64),
                        ("host_block", host_block, torch.int64),
                        ("minimum_ptrs", minimum_ptrs, torch.int64),
                        ("maximum_ptrs", maximum_ptrs, torch.int64),
                        ("summary_ptrs", summary_ptrs, torch.int64)):
        if t is None:
            limits.append(None)
            continue
        if t.dtype != dt or t.shape != (batch,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dt} tensor of {batch} entries")
        limits.append(t.data_ptr())
    # rows of a chunk adjacent (copied when they are not); any distance between chunks
    row = config.kv_heads * config.head_dim
    strides = k.stride()
    if strides != v.stride() or strides[3] != 1 or strides[2] != config.head_dim or \
            (strides[1] != row and tokens > 1):
        k, v = k.contiguous(), v.contiguous()
        strides = (tokens * row,)
    with _lib.on_device(index):
        status = _lib.load().hs_append_quantized(
            batch, tokens, k.data_ptr(), v.data_ptr(), strides[0], _lib.dtype_code(k.dtype),
            *limits[:3], pool.data_ptr(), blocks, limits[3],
            None if host is None else host.data_ptr(),
            0 if host is None else host.tensor.shape[0], *limits[4:], config.kv_heads,
            config.head_dim, config.page_size, _lib.status_pointer(index),
            _lib.raw_stream(index))
    if status:
        _lib.check(status)


def held_values(k, v, config, dtype=None):
    """The values that K and V rows [B, T, Hkv, D] will be held as, in `dtype` (theirs without):
    [2, B, T, Hkv, D] (exact in bfloat16 and float32; those of float16 rows may leave its
    range). Drafted rows that are not appended yet are attended to as those, so that a
    drafted turn computes what the plain turns after it will."""
    batch, tokens = k.shape[:2]
    page = replace(config, gpu_pages=max(1, batch), page_size=max(1, tokens))
    pool = k.new_empty((batch, *page.page_shape), dtype=torch.uint8)
    within = torch.zeros(batch, dtype=torch.int32, device=k.device)
    blocks = torch.arange(batch, device=k.device)
    append_quantized(k, v, within, torch.full_like(within, tokens), blocks, pool, None, None,
                     None, page)
    rows = torch.arange(batch * tokens, device=k.device).view(batch, tokens)
    return read_quantized(pool, rows, page, k.dtype if dtype is None else dtype)


def read_quantized(pool, rows, config, dtype=torch.bfloat16):
    """The values of physical rows of a pool held in 8 bits: K and V as a new
    [2, *rows.shape, Hkv, D] of `dtype`, rounded to it once (they are exact in
    bfloat16 and float32). rows: int64 of any shape; a negative row gives zeros,
    one beyond the pool too, and raises the device flag. Runs on the current
    stream."""
    index = _lib.one_device(pool, rows)
    blocks = check_pool(pool, config)
    if rows.dtype != torch.int64:
        raise ValueError("rows must be int64")
    if dtype not in _VALUES:
        raise ValueError(f"unsupported element type {dtype}")
    rows = rows.contiguous()
    out = pool.new_empty((2, *rows.shape, config.kv_heads, config.head_dim), dtype=dtype)
    with _lib.on_device(index):
        status = _lib.load().hs_read_quantized(
            pool.data_ptr(), blocks, rows.data_ptr(), rows.numel(), out.data_ptr(),
            _lib.dtype_code(dtype), config.kv_heads, config.head_dim, config.page_size,
            _lib.status_pointer(index), _lib.raw_stream(index))
    if status:
        _lib.check(status)
    return out


def attend_quantized(query, pool, rows, config, counts=None):
    """Decode attention of query [B, Hq, D] over physical rows of a pool held in 8
    bits: ``attend_rows`` for a batch.

    rows: int64 [B, K], shared by the heads of a request, or [B, Hq, K]; -1 entries
    are masked. counts: int32 [B], leading rows to read (all K without). A head
    that sees no row gets zeros. Heads of the query adjacent, any distance between
    requests. Returns a new [B, Hq, D] of the query's dtype; sums are fp32. Runs on
    the current stream.
    """
    index = _lib.one_device(query, pool, rows, counts)
    blocks = check_pool(pool, config)
    shape, kv_heads = query.shape, config.kv_heads
    if len(shape) != 3 or shape[2] != config.head_dim:
        raise ValueError("query must be [batch, heads, head_dim]")
    batch, q_heads, dim = shape
    if q_heads < 1 or q_heads % kv_heads:
        raise ValueError("query GQA/device mismatch")
    code = _lib.dtype_code(query.dtype)
    wanted = rows.shape
    if rows.dtype != torch.int64 or wanted[:-1] not in ((batch,), (batch, q_heads)):
        raise ValueError("rows must be int64 [batch, rows] or [batch, heads, rows]")
    limit = None
    if counts is not None:
        if counts.dtype != torch.int32 or counts.shape != (batch,) or not counts.is_contiguous():
            raise ValueError("counts must be contiguous int32 [batch]")
        limit = counts.data_ptr()
    q_batch, head, inner = query.stride()
    if inner != 1 or head != dim:
        query = query.contiguous()
        q_batch = q_heads * dim
    count = wanted[-1]
    if rows.stride(-1) != 1 and count > 1:
        rows = rows.contiguous()
    row_batch, row_head = rows.stride(0), 0 if len(wanted) == 2 else rows.stride(1)
    if len(wanted) == 3 and q_heads == 1:
        row_head = 0
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    lib = _lib.load()
    with _lib.on_device(index):
        nbytes = lib.hs_attend_quantized_workspace_bytes(batch, 1, code, q_heads, kv_heads, dim,
                                                         count)
        ws = query.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        status = lib.hs_attend_quantized(
            batch, query.data_ptr(), q_batch, code, pool.data_ptr(), blocks, rows.data_ptr(),
            row_batch, row_head, count, limit, out.data_ptr(), q_heads, kv_heads, dim,
            config.page_size, _lib.ptr(ws), nbytes, _lib.status_pointer(index),
            _lib.raw_stream(index))
    if status:
        _lib.check(status)
    return out
