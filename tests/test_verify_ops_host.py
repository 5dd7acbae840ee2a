"""The verification operators' C ABI: every declared symbol is exported and bad
arguments are refused on the host, before any device work (no GPU needed)."""

import ctypes
import re
from pathlib import Path

import pytest
import torch

from hisparse_b200 import _lib

HEADER = Path(__file__).resolve().parent.parent / "include" / "hisparse_verify.h"
D = 256  # a dummy non-null pointer value: never dereferenced on these paths
BAD, UNSUPPORTED = _lib.HS_ERR_INVALID_ARGUMENT, _lib.HS_ERR_UNSUPPORTED


def test_every_declared_symbol_is_exported():
    names = re.findall(r"^HS_API\s+[\w\s\*]*?\b(hs_\w+)\s*\(", HEADER.read_text(), flags=re.M)
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    assert set(names) == set(_lib._VERIFY_SIGNATURES)
    for name in names:
        assert hasattr(lib, name), name


def norm_rope(tokens=1, hq=8, hkv=2, dim=32, dtype=_lib.HS_BFLOAT16, q=D, pos=D,
              pos_dtype=_lib.HS_INT32, eps=1e-6):
    return _lib.load().hs_qk_norm_rope(tokens, q, hq * dim, dim, hq, D, hkv * dim, dim, hkv, dim,
                                       dtype, pos, pos_dtype, D, None, None, eps, D, D, None)


def test_norm_rope_validation():
    assert norm_rope(tokens=-1) == BAD
    assert norm_rope(hq=0) == BAD
    assert norm_rope(dim=33) == BAD
    assert norm_rope(dim=258) == UNSUPPORTED
    assert norm_rope(dtype=9) == BAD
    assert norm_rope(q=None) == BAD and b"null" in _lib.load().hs_last_error()
    assert norm_rope(pos_dtype=_lib.HS_FLOAT32) == BAD
    assert norm_rope(eps=float("nan")) == BAD
    assert norm_rope(tokens=0, q=None) == _lib.HS_OK


def logprobs(rows=1, logits=D, dtype=_lib.HS_FLOAT32, vocab=100, tokens=D,
             tokens_dtype=_lib.HS_INT64, given=1, out=D, top=4, top_out=D):
    return _lib.load().hs_token_logprobs(rows, logits, vocab, dtype, vocab, tokens, tokens_dtype,
                                         given, out, D, top, top_out, top_out, None, None)


def test_logprobs_validation():
    assert logprobs(rows=-1) == BAD
    assert logprobs(vocab=0) == BAD
    assert logprobs(vocab=2 ** 31) == BAD
    assert logprobs(top=101) == BAD
    assert logprobs(top=33) == UNSUPPORTED
    assert logprobs(given=-1) == BAD
    assert logprobs(tokens=None) == BAD
    assert logprobs(tokens_dtype=_lib.HS_FLOAT32) == BAD
    assert logprobs(top_out=None) == BAD
    assert logprobs(dtype=_lib.HS_INT32) == BAD
    assert logprobs(rows=0, logits=None) == _lib.HS_OK


def tree(batch=2, nodes=4, q=D, dtype=_lib.HS_BFLOAT16, mask=D, pool=D, rows=D, count=64, hq=8,
         hkv=2, dim=32, page=16, ws=None, ws_bytes=0):
    return _lib.load().hs_attend_tree(batch, nodes, q, 4 * hq * dim, hq * dim, D, D, 4 * hkv * dim,
                                      hkv * dim, dtype, mask, None, pool, 100, rows, count, count,
                                      None, D, hq, hkv, dim, page, ws, ws_bytes, None, None)


def test_tree_validation():
    lib = _lib.load()
    assert tree(batch=-1) == BAD
    assert tree(hq=7) == BAD and lib.hs_last_error() == b"query GQA/device mismatch"
    assert tree(nodes=65) == UNSUPPORTED
    assert tree(dim=257) == UNSUPPORTED
    assert tree(dim=0) == BAD
    assert tree(dtype=_lib.HS_INT32) == BAD
    assert tree(mask=None) == BAD
    assert tree(rows=None) == BAD
    assert tree(page=0) == BAD
    assert tree(count=-1) == BAD
    need = lib.hs_attend_tree_workspace_bytes(1, 8, 32, 8, 128, 32768, _lib.HS_BFLOAT16)
    assert need > 0
    assert tree(batch=1, nodes=8, hq=32, hkv=8, dim=128, count=32768) == _lib.HS_ERR_WORKSPACE
    assert tree(batch=1, nodes=8, hq=32, hkv=8, dim=128, count=32768, ws=D,
                ws_bytes=need - 1) == _lib.HS_ERR_WORKSPACE
    assert tree(batch=1, nodes=8, hq=32, hkv=8, dim=128, count=32768, ws=D + 8,
                ws_bytes=need) == _lib.HS_ERR_WORKSPACE
    assert b"16-byte" in lib.hs_last_error()
    assert tree(batch=0, q=None) == _lib.HS_OK


def test_operators_refuse_cpu_tensors():
    from hisparse_b200 import CacheConfig, attend_tree, qk_norm_rope, token_logprobs

    x, p = torch.zeros(2, 2, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(x, x, p, torch.ones(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="CUDA"):
        t = torch.zeros(1, 2, 2, 8)
        attend_tree(t, t, t, torch.zeros(1, 2, dtype=torch.int64), torch.zeros(4, 2, 16, 2, 8),
                    torch.zeros(1, 3, dtype=torch.int64), CacheConfig(head_dim=8))
