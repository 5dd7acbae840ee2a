"""A cache held in 8 bits, on the CPU: the C ABI's symbols and refusals, the operators'
argument checks, the configuration, and the tests' own 64-bit forms."""

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import quantized_reference as ref
from hisparse_b200 import (CacheConfig, _lib, append_quantized, attend_quantized,
                           read_quantized)

HEADER = Path(__file__).resolve().parent.parent / "include" / "hisparse_quantized.h"
E4M3 = torch.float8_e4m3fn


def test_every_declared_symbol_is_exported():
    names = re.findall(r"^HS_API\s+[\w\s\*]*?\b(hs_\w+)\s*\(", HEADER.read_text(), flags=re.M)
    assert len(names) == 7 and set(names) == set(_lib._QUANTIZED_SIGNATURES)
    lib = ctypes.CDLL(str(_lib.LIB_PATH))
    for name in names:
        assert hasattr(lib, name), name


@pytest.mark.parametrize("heads,dim", [(1, 1), (2, 32), (8, 128), (4, 128), (3, 7), (1, 256)])
def test_row_bytes(heads, dim):
    config = CacheConfig(kv_heads=heads, head_dim=dim, dtype=E4M3)
    assert config.row_bytes == ref.row_bytes(heads, dim)
    assert _lib.load().hs_quantized_row_bytes(heads, dim) == config.row_bytes
    assert config.row_bytes % 32 == 0 and 0 <= config.row_bytes - heads * (dim + 1) < 32
    assert config.page_shape == (2, 16, config.row_bytes)
    assert config.storage_dtype == torch.uint8 and config.metadata_dtype == torch.bfloat16


def test_configurations():
    plain = CacheConfig(dtype=torch.float16)
    assert not plain.quantized and plain.page_shape == (2, 16, 2, 32)
    assert plain.storage_dtype == plain.metadata_dtype == torch.float16
    with pytest.raises(ValueError, match="head_dim up to 256"):
        CacheConfig(head_dim=257, dtype=E4M3)
    with pytest.raises(ValueError, match="KV dtype"):
        CacheConfig(dtype=torch.float8_e5m2)
    assert _lib.load().hs_quantized_row_bytes(0, 8) == 0


def test_host_side_validation_needs_no_device():
    lib = _lib.load()
    bad, unsupported, workspace = (_lib.HS_ERR_INVALID_ARGUMENT, _lib.HS_ERR_UNSUPPORTED,
                                   _lib.HS_ERR_WORKSPACE)

    def append(batch=1, dtype=_lib.HS_BFLOAT16, heads=2, dim=32, page=16, k=16):
        return lib.hs_append_quantized(batch, 1, k, 16, 64, dtype, 16, 16, 16, 16, 4, 16, None, 0,
                                       16, 16, 16, heads, dim, page, None, None)

    assert append(batch=0) == _lib.HS_OK
    assert append(batch=-1) == append(heads=0) == append(page=0) == append(dtype=7) == bad
    assert append(k=None) == bad
    # bounds without the mean
    assert lib.hs_append_quantized(1, 1, 16, 16, 64, 0, 16, 16, 16, 16, 4, 16, None, 0, 16, 16,
                                   None, 2, 32, 16, None, None) == bad
    assert append(dim=257) == append(batch=65536) == append(heads=1 << 20) == unsupported

    def read(count=4, dtype=_lib.HS_FLOAT32, dim=32, pool=16):
        return lib.hs_read_quantized(pool, 4, 16, count, 16, dtype, 2, dim, 16, None, None)

    assert read(count=0) == _lib.HS_OK
    assert read(count=-1) == read(dtype=5) == read(pool=None) == read(pool=8) == bad
    assert read(dim=257) == unsupported

    def attend(batch=1, q_heads=4, dim=32, count=4096, dtype=_lib.HS_FLOAT32, ws=16, nbytes=1 << 30,
               pool=16):
        return lib.hs_attend_quantized(batch, 16, 128, dtype, pool, 4, 16, count, 0, count, None,
                                       16, q_heads, 2, dim, 16, ws, nbytes, None, None)

    assert attend(batch=0) == _lib.HS_OK
    assert attend(q_heads=5) == attend(count=-1) == attend(dtype=9) == attend(pool=None) == bad
    assert attend(pool=24) == bad
    assert attend(dim=257) == attend(batch=65536) == unsupported
    assert lib.hs_attend_quantized_workspace_bytes(1, 1, _lib.HS_FLOAT32, 4, 2, 32, 4096) > 0
    assert attend(ws=None) == attend(nbytes=8) == attend(ws=8) == workspace

    def phase(phase=0, counts_n=1, nbytes=1 << 30):
        return lib.hs_attend_quantized_phase(1, 16, 128, _lib.HS_FLOAT32, 16, 4, 16, 64, 64, 16, 3,
                                             0, counts_n, phase, 4, 2, 32, 16, 16, nbytes, None,
                                             None)

    assert phase(phase=2) == phase(phase=-1) == phase(counts_n=-1) == bad
    assert phase(nbytes=8) == workspace
    assert lib.hs_attend_quantized_merge(1, 3, 16, 0, 4, 2, 32, 64, 16, 1 << 30, None) == bad
    assert lib.hs_attend_quantized_merge(1, 2, None, 0, 4, 2, 32, 64, 16, 1 << 30, None) == bad
    assert lib.hs_attend_quantized_merge(1, 2, 16, 0, 4, 2, 32, 64, 16, 8, None) == workspace
    sizes = _lib.HS_FLOAT32, 4, 2, 32, 4096
    assert lib.hs_attend_quantized_workspace_bytes(2, 2, *sizes) >= \
        2 * lib.hs_attend_quantized_workspace_bytes(2, 1, *sizes) > 0


def test_operators_refuse_cpu_tensors():
    config = CacheConfig(kv_heads=2, head_dim=8, page_size=4, dtype=E4M3)
    pool = torch.zeros((3, *config.page_shape), dtype=torch.uint8)
    rows = torch.zeros((1, 4), dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        read_quantized(pool, rows, config)
    with pytest.raises(ValueError, match="CUDA"):
        attend_quantized(torch.zeros(1, 4, 8), pool, rows, config)
    with pytest.raises(ValueError, match="CUDA"):
        append_quantized(torch.zeros(1, 1, 2, 8), torch.zeros(1, 1, 2, 8), rows[0, :1].int(),
                         rows[0, :1].int(), rows[0, :1], pool, rows[0, :1], rows[0, :1],
                         rows[0, :1], config)


def test_reference_encoding_is_the_types():
    """The tests' codes against torch's e4m3, over every number and around every border."""
    numbers = ref.NUMBERS[:127]
    assert np.array_equal(torch.arange(127, dtype=torch.uint8).view(E4M3).double().numpy(), numbers)
    between = (numbers[1:] + numbers[:-1]) / 2
    x = np.concatenate([numbers, between, np.nextafter(between, 0), np.nextafter(between, 999)])
    x = x.astype(np.float32).astype(np.float64)
    x = np.concatenate([x, -x])
    expected = torch.from_numpy(x).float().to(E4M3).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(x), expected)
    assert ref.exponent(np.array([448.0])) == 0 and ref.exponent(np.array([448.001])) == 1
    assert ref.exponent(np.array([0.0])) == ref.exponent(np.array([1e-38])) == -100
