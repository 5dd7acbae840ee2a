"""Calls at the edges of what the verification operators' documentation allows."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def flags():
    from hisparse_b200 import _lib

    return _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("width", [0, 40])
def test_tree_marks_of_values_that_are_not_finite(dtype, dim, width):
    """The marks of such values are written by the warps that copy them and read by the
    softmax warps as soon as the products are done. The shortest way from one to the
    other: one or two blocks of keys, the value in the last one, on every SM at once."""
    from hisparse_b200 import attend_tree, tree_mask
    from test_gpu_verify_ops import tree_inputs

    batch, nodes = 96, 30
    (q, k, v), _, pool, rows, config = tree_inputs(batch, nodes, 8, 4, dim, 16, width, dtype, 51)
    mask = tree_mask([[-1] + [(t - 1) // 2 for t in range(1, nodes)]] * batch, DEV)
    clean = attend_tree(q, k, v, mask, pool, rows, config)
    v[:, 29, 3, dim - 1] = math.inf  # a leaf: only it sees its value
    v[:, 0, 1, 0] = math.nan         # the root: every node does
    for _ in range(20):
        got = attend_tree(q, k, v, mask, pool, rows, config)
        assert bool((got[:, 29, 6:, dim - 1] == math.inf).all())
        assert bool(got[:, :, 2:4, 0].isnan().all())
        same = torch.ones_like(got, dtype=torch.bool)
        same[:, 29, 6:, dim - 1] = False
        same[:, :, 2:4, 0] = False
        assert torch.equal(got[same], clean[same])
    assert not flags()
