"""Per-head norms of queries and keys with the position rotation, in one pass
(``hs_qk_norm_rope``).

The decoder of nano_hisparse/model.py:136-155 rotates queries and keys with a
chain of torch calls and has no per-head norms; models that normalise each
query and key head before the rotation take both through this operator
(``DecoderConfig.qk_norm``).
"""

from __future__ import annotations

import torch

from . import _lib


def rope_frequencies(head_dim: int, theta: float, device="cuda") -> torch.Tensor:
    """theta^(-2i/head_dim) for i < head_dim / 2, in fp64 (the angles of far
    positions lose their fraction of a turn with fp32 frequencies)."""
    if head_dim < 2 or head_dim % 2:
        raise ValueError("head_dim must be even")
    exponent = torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim
    return float(theta) ** -exponent


def _check_heads(name, x, tokens, head_dim, dtype):
    if x.ndim != 3 or x.shape[0] != tokens or x.shape[2] != head_dim or x.shape[1] < 1:
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    if x.dtype != dtype:
        raise ValueError("query, key and weights must have one dtype")
    # an inner stride other than 1 is laid out anew; any other stride is read in place
    return x if x.stride(2) == 1 else x.contiguous()


def qk_norm_rope(query, key, positions, inv_freq, query_weight=None, key_weight=None, eps=1e-6):
    """RMS-normalise every query and key head (with a weight; without one the
    norm is left out), then rotate the pairs (i, i + head_dim / 2) by
    positions * inv_freq[i].

    query [N, Hq, D] and key [N, Hkv, D]: CUDA, one dtype (fp32, fp16, bf16),
    any token and head stride (views of a fused projection need no copy), D
    even and at most 256. positions: int32 or int64 [N]. inv_freq: fp64
    [D / 2], see ``rope_frequencies``. query_weight / key_weight: [D] of the
    same dtype. Returns new contiguous (query, key); fp32 arithmetic with one
    rounding. Runs on the current stream.
    """
    _lib.require_cuda(query, key, positions, inv_freq, query_weight, key_weight)
    if query.ndim != 3:
        raise ValueError("query must be [tokens, heads, head_dim]")
    tokens, q_heads, dim = query.shape
    query = _check_heads("query", query, tokens, dim, query.dtype)
    key = _check_heads("key", key, tokens, dim, query.dtype)
    if dim < 2 or dim % 2:
        raise ValueError("head_dim must be even")
    if positions.shape != (tokens,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64 [tokens]")
    if inv_freq.shape != (dim // 2,) or inv_freq.dtype != torch.float64:
        raise ValueError("inv_freq must be float64 [head_dim / 2]")
    for w in (query_weight, key_weight):
        if w is not None and (w.shape != (dim,) or w.dtype != query.dtype):
            raise ValueError("norm weights must be [head_dim] of the query's dtype")
    device = query.device
    for t in (key, positions, inv_freq, query_weight, key_weight):
        if t is not None and t.device != device:
            raise ValueError("all tensors must be on one device")
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    if query_weight is not None:
        query_weight = query_weight.contiguous()
    if key_weight is not None:
        key_weight = key_weight.contiguous()
    query_out = torch.empty((tokens, q_heads, dim), dtype=query.dtype, device=device)
    key_out = torch.empty((tokens, key.shape[1], dim), dtype=query.dtype, device=device)
    with _lib.on_device(device):
        _lib.check(_lib.load().hs_qk_norm_rope(
            tokens, query.data_ptr(), query.stride(0), query.stride(1), q_heads, key.data_ptr(),
            key.stride(0), key.stride(1), key.shape[1], dim, _lib.dtype_code(query.dtype),
            positions.data_ptr(),
            _lib.HS_INT64 if positions.dtype == torch.int64 else _lib.HS_INT32,
            inv_freq.data_ptr(), _lib.ptr(query_weight), _lib.ptr(key_weight), eps,
            query_out.data_ptr(), key_out.data_ptr(), _lib.stream_of(device)))
    return query_out, key_out
