"""Log probabilities of given tokens, the distribution's entropy and its
largest alternatives, in one pass over the logits (``hs_token_logprobs``).

The reference engine takes the argmax of fp32 logits only
(nano_hisparse/model.py:179, engine.py:90-120); scoring drafted or given
tokens needs the normaliser as well.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_TOKENS = {torch.int32: _lib.HS_INT32, torch.int64: _lib.HS_INT64}


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # fp32, the shape of the given tokens ([N, 0] without)
    entropy: torch.Tensor       # fp32 [N], nats
    top_logprobs: torch.Tensor  # fp32 [N, top], largest first
    top_tokens: torch.Tensor    # int64 [N, top]; equal logits by the lower token


def token_logprobs(logits, tokens=None, top=0) -> TokenLogprobs:
    """logits: CUDA [N, V] (fp32, fp16, bf16; any row stride). tokens: int32 or
    int64 [N] or [N, C]; a negative token is padding (log probability 0), one
    past the vocabulary gives NaN and raises the device flag. top: how many of
    the largest entries to return (at most 32). All results are fp32 sums over
    the given values; -inf logits have probability 0, and a row with nothing
    above -inf has log probabilities -inf and entropy 0. Runs on the current
    stream."""
    index = _lib.one_device(logits, tokens)
    shape = logits.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError("logits must be [rows, vocab]")
    rows, vocab = shape
    if not 0 <= top <= vocab:
        raise ValueError("top must be between 0 and the vocabulary size")
    shape, given, code, address = (rows, 0), 0, _lib.HS_INT64, None
    if tokens is not None:
        shape, code = tokens.shape, _TOKENS.get(tokens.dtype)
        if code is None or len(shape) not in (1, 2) or shape[0] != rows:
            raise ValueError("tokens must be int32 or int64 [rows] or [rows, given]")
        given = 1 if len(shape) == 1 else shape[1]
        tokens = tokens.contiguous()
        address = tokens.data_ptr()
    row_stride, inner = logits.stride()
    if inner != 1:
        logits = logits.contiguous()
        row_stride = vocab
    # like one another where the shapes agree: that is made faster than a new shape
    if tokens is None:
        logprobs = logits.new_empty(shape, dtype=torch.float32)
    else:
        logprobs = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprobs) if len(shape) == 1 else \
        logits.new_empty(rows, dtype=torch.float32)
    top_tokens = logits.new_empty((rows, top), dtype=torch.int64)
    top_logprobs = torch.empty_like(top_tokens, dtype=torch.float32)
    with _lib.on_device(index):
        status = _lib.load().hs_token_logprobs(
            rows, logits.data_ptr(), row_stride, _lib.dtype_code(logits.dtype), vocab, address,
            code, given, logprobs.data_ptr(), entropy.data_ptr(), top, top_logprobs.data_ptr(),
            top_tokens.data_ptr(), _lib.status_pointer(index), _lib.raw_stream(index))
    if status:
        _lib.check(status)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)
