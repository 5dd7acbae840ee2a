"""The bounds of the attention tests over a cache held in 8 bits, on the CPU: what they are there
to find exceeds them."""

import numpy as np
import pytest
import torch

import quantized_bounds as bounds
import quantized_reference as ref
from test_gpu_quantized_exact import CANCELLING, FLAT, cancelling, flat

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rounded(x, dtype):
    return torch.from_numpy(x).to(dtype).double().numpy()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", FLAT)
def test_a_missing_row_is_found(dtype, case):
    """Without its row of median weight, or without any 32 neighbouring ones, every request's
    result leaves its bound."""
    query, pool, rows = flat(*case, dtype)
    heads, dim = case[2], case[3]
    query, rows = query[:1].double().numpy(), rows[:1]
    out, bound = bounds.attend(query, pool, rows, heads, dtype)
    assert np.all(np.abs(rounded(out, dtype) - out) <= bound)
    middle = rows.shape[1] // 2
    for gone in (slice(middle, middle + 1), slice(0, 32), slice(rows.shape[1] - 32, None)):
        less = rows.copy()
        less[:, gone] = -1
        other, _ = bounds.attend(query, pool, less, heads, dtype)
        assert np.any(np.abs(rounded(other, dtype) - out) > bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CANCELLING)
def test_weights_in_one_fp16_number_are_found(dtype, case):
    query, pool, rows, some = cancelling(*case, dtype)
    _, _, heads, dim, _ = case
    q = query.double().numpy()
    out, bound = bounds.attend(q, pool, rows, heads, dtype)
    group, found = case[1] // heads, False
    for h in some:
        kh = h // group
        k, v = (ref.values(ref.row_records(pool, rows[0], plane), heads, dim)[:, kh]
                for plane in range(2))
        e = ref.row_records(pool, rows[0], 1)[:, heads * dim + kh].astype(int) - 127
        s = k @ q[0, h] / np.sqrt(dim) * np.log2(np.e)
        lifted = np.exp2(s + e - (s + e).max() + 7)
        total = np.exp2(s - (s + e).max() + 7).sum()
        for bits, weights in (("one", lifted.astype(np.float16).astype(float)),
                              ("two", lifted.astype(np.float16).astype(float) + (
                                  lifted - lifted.astype(np.float16)).astype(np.float16))):
            result = rounded(weights @ (v * np.exp2(-e.astype(float))[:, None]) / total, dtype)
            outside = np.any(np.abs(result - out[0, h]) > bound[0, h])
            assert bits == "one" or not outside
            found |= bits == "one" and outside
    assert found
