"""Attention of a tree of drafted tokens over selected cache rows and over the
tree itself (``hs_attend_tree``).

``attend_rows`` (nano_hisparse/row_kernels.py:116-135) serves one new token of
a request whose K/V row is in the pool already. Here a request has up to 64
drafted tokens (nodes) whose K/V are the step's own tensors and enter the
cache only if they are accepted; all of them share the request's physical
rows, and each also sees the nodes that its mask names (a drafted tree: its
ancestors and itself).
"""

from __future__ import annotations

import torch

from . import _lib

MAX_NODES = 64


def tree_mask(parents, device="cuda") -> torch.Tensor:
    """int64 [B, T] masks of drafted trees. parents[b] lists each node's parent
    in request b's tree (a lower index, or -1 for a node with none); shorter
    trees are padded with nodes that see nothing. Bit j of mask[b, t] is set
    when j is t or an ancestor of t."""
    width = max((len(p) for p in parents), default=0)
    if width > MAX_NODES:
        raise ValueError(f"a tree has more than {MAX_NODES} nodes")
    out = []
    for tree in parents:
        masks = []
        for t, parent in enumerate(tree):
            if not -1 <= parent < t:
                raise ValueError("a node's parent must come before it")
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << t)
        masks += [0] * (width - len(tree))
        out.append([m - (1 << 64) if m >> 63 else m for m in masks])
    return torch.tensor(out, dtype=torch.int64).view(len(out), width).to(device)


def attend_tree(query, key, value, mask, pool, rows, config, counts=None, nodes=None):
    """Attention of query [B, T, Hq, D] over pool rows and the nodes' key/value
    [B, T, Hkv, D]; T <= 64.

    mask: int64 [B, T], bit j of mask[b, t] lets node t see node j. pool and
    config: as ``attend_rows``. rows: int64 [B, K] physical rows of each
    request, -1 entries masked; every node sees all of them. counts: int32 [B],
    leading rows to read (all K without). nodes: int32 [B], nodes of each
    request's tree (all T without); the results of nodes past it are zero, and
    nothing of theirs is read. A node that sees nothing gets zeros. One dtype
    throughout; any batch and node stride of query, key and value with adjacent
    heads. Returns a new [B, T, Hq, D]. Runs on the current stream.
    """
    index = _lib.one_device(query, key, value, mask, pool, rows, counts, nodes)
    shape, dtype, kv_heads = query.shape, query.dtype, config.kv_heads
    if len(shape) != 4 or shape[3] != config.head_dim:
        raise ValueError("query must be [batch, nodes, heads, head_dim]")
    batch, width, q_heads, dim = shape
    if q_heads < 1 or q_heads % kv_heads:
        raise ValueError("query GQA/device mismatch")
    if width > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} nodes are supported")
    kv_shape = (batch, width, kv_heads, dim)
    if key.shape != kv_shape or value.shape != kv_shape:
        raise ValueError("key and value must be [batch, nodes, kv_heads, head_dim]")
    blocks, *block = pool.shape
    if block != [2, config.page_size, kv_heads, dim] or not pool.is_contiguous():
        raise ValueError("pool must be contiguous [blocks, 2, page_size, kv_heads, head_dim]")
    if not dtype == key.dtype == value.dtype == pool.dtype:
        raise ValueError("query, key, value and pool must have one dtype")
    if mask.shape != (batch, width) or mask.dtype != torch.int64:
        raise ValueError("mask must be int64 [batch, nodes]")
    rows_shape = rows.shape
    if len(rows_shape) != 2 or rows_shape[0] != batch or rows.dtype != torch.int64:
        raise ValueError("rows must be int64 [batch, rows]")
    limits = []  # addresses of counts and nodes
    for name, t in (("counts", counts), ("nodes", nodes)):
        if t is None:
            limits.append(None)
            continue
        if t.dtype != torch.int32 or t.shape != (batch,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [batch]")
        limits.append(t.data_ptr())
    # heads of a node adjacent (copied when they are not); batch and node strides as they are
    q_batch, q_node, head, inner = query.stride()
    if inner != 1 or head != dim:
        query = query.contiguous()
        q_batch, q_node, _, _ = query.stride()
    strides = key.stride()
    if strides != value.stride() or strides[3] != 1 or strides[2] != dim:
        key, value = key.contiguous(), value.contiguous()
        strides = (width * kv_heads * dim, kv_heads * dim)
    mask, count = mask.contiguous(), rows_shape[1]
    row_stride, inner = rows.stride()
    if inner != 1 and count > 1:
        rows = rows.contiguous()
        row_stride = count
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    lib, code = _lib.load(), _lib.dtype_code(dtype)
    with _lib.on_device(index):
        nbytes = lib.hs_attend_tree_workspace_bytes(batch, width, q_heads, kv_heads, dim, count,
                                                    code)
        ws = query.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        status = lib.hs_attend_tree(
            batch, width, query.data_ptr(), q_batch, q_node, key.data_ptr(), value.data_ptr(),
            strides[0], strides[1], code, mask.data_ptr(), limits[1], pool.data_ptr(), blocks,
            rows.data_ptr(), row_stride, count, limits[0], out.data_ptr(), q_heads, kv_heads, dim,
            config.page_size, _lib.ptr(ws), nbytes, _lib.status_pointer(index),
            _lib.raw_stream(index))
    if status:
        _lib.check(status)
    return out
