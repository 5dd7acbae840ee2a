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

_POSITIONS = {torch.int32: _lib.HS_INT32, torch.int64: _lib.HS_INT64}


def rope_frequencies(head_dim: int, theta: float, device="cuda") -> torch.Tensor:
    """theta^(-2i/head_dim) for i < head_dim / 2, in fp64 (the angles of far
    positions lose their fraction of a turn with fp32 frequencies)."""
    if head_dim < 2 or head_dim % 2:
        raise ValueError("head_dim must be even")
    exponent = torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim
    return float(theta) ** -exponent


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
    index = _lib.one_device(query, key, positions, inv_freq, query_weight, key_weight)
    dtype, shape, key_shape = query.dtype, query.shape, key.shape
    if len(shape) != 3 or shape[1] < 1:
        raise ValueError("query must be [tokens, heads, head_dim]")
    tokens, q_heads, dim = shape
    if len(key_shape) != 3 or key_shape[0] != tokens or key_shape[2] != dim or key_shape[1] < 1:
        raise ValueError("key must be [tokens, heads, head_dim]")
    if key.dtype != dtype:
        raise ValueError("query, key and weights must have one dtype")
    if dim < 2 or dim % 2:
        raise ValueError("head_dim must be even")
    code = _POSITIONS.get(positions.dtype)
    if code is None or positions.shape != (tokens,):
        raise ValueError("positions must be int32 or int64 [tokens]")
    if inv_freq.dtype != torch.float64 or inv_freq.shape != (dim // 2,):
        raise ValueError("inv_freq must be float64 [head_dim / 2]")
    q_weight = k_weight = None  # addresses
    if query_weight is not None:
        if query_weight.dtype != dtype or query_weight.shape != (dim,):
            raise ValueError("norm weights must be [head_dim] of the query's dtype")
        query_weight = query_weight.contiguous()
        q_weight = query_weight.data_ptr()
    if key_weight is not None:
        if key_weight.dtype != dtype or key_weight.shape != (dim,):
            raise ValueError("norm weights must be [head_dim] of the query's dtype")
        key_weight = key_weight.contiguous()
        k_weight = key_weight.data_ptr()
    # an inner stride other than 1 is laid out anew; any other stride is read in place
    q_token, q_head, inner = query.stride()
    if inner != 1:
        query = query.contiguous()
        q_token, q_head, _ = query.stride()
    k_token, k_head, inner = key.stride()
    if inner != 1:
        key = key.contiguous()
        k_token, k_head, _ = key.stride()
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    query_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    key_out = torch.empty_like(key, memory_format=torch.contiguous_format)
    with _lib.on_device(index):
        status = _lib.load().hs_qk_norm_rope(
            tokens, query.data_ptr(), q_token, q_head, q_heads, key.data_ptr(), k_token, k_head,
            key_shape[1], dim, _lib.dtype_code(dtype), positions.data_ptr(), code,
            inv_freq.data_ptr(), q_weight, k_weight, eps, query_out.data_ptr(),
            key_out.data_ptr(), _lib.raw_stream(index))
    if status:
        _lib.check(status)
    return query_out, key_out
