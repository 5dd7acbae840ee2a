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


def _heads_adjacent(x):
    """x [B, T, H, D] with the heads of a node adjacent (copied when they are not)."""
    return x if x.stride(3) == 1 and x.stride(2) == x.shape[3] else x.contiguous()


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
    if query.ndim != 4 or query.shape[3] != config.head_dim:
        raise ValueError("query must be [batch, nodes, heads, head_dim]")
    batch, width, q_heads, dim = query.shape
    if q_heads < 1 or q_heads % config.kv_heads:
        raise ValueError("query GQA/device mismatch")
    if width > MAX_NODES:
        raise ValueError(f"at most {MAX_NODES} nodes are supported")
    kv_shape = (batch, width, config.kv_heads, dim)
    if key.shape != kv_shape or value.shape != kv_shape:
        raise ValueError("key and value must be [batch, nodes, kv_heads, head_dim]")
    if pool.ndim != 5 or pool.shape[1:] != (2, config.page_size, config.kv_heads, dim) \
            or not pool.is_contiguous():
        raise ValueError("pool must be contiguous [blocks, 2, page_size, kv_heads, head_dim]")
    if not query.dtype == key.dtype == value.dtype == pool.dtype:
        raise ValueError("query, key, value and pool must have one dtype")
    if mask.shape != (batch, width) or mask.dtype != torch.int64:
        raise ValueError("mask must be int64 [batch, nodes]")
    if rows.ndim != 2 or rows.shape[0] != batch or rows.dtype != torch.int64:
        raise ValueError("rows must be int64 [batch, rows]")
    for name, t in (("counts", counts), ("nodes", nodes)):
        if t is not None and (t.shape != (batch,) or t.dtype != torch.int32
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous int32 [batch]")
    query, key, value, mask = (_heads_adjacent(query), _heads_adjacent(key),
                               _heads_adjacent(value), mask.contiguous())
    if key.stride() != value.stride():
        key, value = key.contiguous(), value.contiguous()
    if rows.stride(1) != 1 and rows.shape[1] > 1:
        rows = rows.contiguous()
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    lib, code, count = _lib.load(), _lib.dtype_code(query.dtype), rows.shape[1]
    q_batch, q_node, _, _ = query.stride()
    kv_batch, kv_node, _, _ = key.stride()
    with _lib.on_device(index):
        nbytes = lib.hs_attend_tree_workspace_bytes(batch, width, q_heads, config.kv_heads, dim,
                                                    count, code)
        ws = _lib.workspace(nbytes, query.device)
        _lib.check(lib.hs_attend_tree(
            batch, width, query.data_ptr(), q_batch, q_node, key.data_ptr(), value.data_ptr(),
            kv_batch, kv_node, code, mask.data_ptr(), _lib.ptr(nodes), pool.data_ptr(),
            pool.shape[0], rows.data_ptr(), rows.stride(0), count, _lib.ptr(counts),
            out.data_ptr(), q_heads, config.kv_heads, dim, config.page_size, _lib.ptr(ws), nbytes,
            _lib.status_pointer(index), _lib.raw_stream(index)))
    return out
