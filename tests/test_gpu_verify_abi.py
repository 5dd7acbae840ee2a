"""Calls of the verification operators' C ABI that the Python wrappers never make."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def tree_call(q, k, v, mask, pool, rows, out, config):
    """hs_attend_tree into `out`, a flat view at any element of a buffer."""
    from hisparse_b200 import _lib

    lib, code = _lib.load(), _lib.dtype_code(q.dtype)
    batch, nodes, hq, dim = q.shape
    hkv, count = k.shape[2], rows.shape[1]
    need = lib.hs_attend_tree_workspace_bytes(batch, nodes, hq, hkv, dim, count, code)
    ws = _lib.workspace(need, DEV)
    _lib.check(lib.hs_attend_tree(
        batch, nodes, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(),
        k.stride(0), k.stride(1), code, mask.data_ptr(), None, pool.data_ptr(), pool.shape[0],
        rows.data_ptr(), rows.stride(0), count, None, out.data_ptr(), hq, hkv, dim,
        config.page_size, _lib.ptr(ws), need, _lib.status_word(DEV).data_ptr(),
        _lib.stream_of(DEV)))
    return need


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("width", [48, 4000])
def test_tree_result_at_any_element(dtype, dim, width):
    """`out` off a 16-byte boundary, with one split (48 rows) and several (4,000): the
    same results as attend_tree's own within its bound, and nothing beside them."""
    from hisparse_b200 import _lib, attend_tree, tree_mask
    from test_gpu_verify_ops import tree_check, tree_inputs

    inputs, parents, pool, rows, config = tree_inputs(2, 5, 8, 2, dim, 16, width, dtype, 41)
    mask = tree_mask(parents, DEV)
    own = attend_tree(*inputs, mask, pool, rows, config)
    for offset in (0, 1, 2, 4, 8):
        buffer = torch.full((own.numel() + 32,), 7.0, dtype=dtype, device=DEV)
        out = buffer[offset:offset + own.numel()]
        need = tree_call(*inputs, mask, pool, rows, out, config)
        assert (need > 0) == (width == 4000)
        tree_check(out.view(own.shape), inputs, mask, pool, rows)
        if out.data_ptr() % 16 == 0 or width == 4000:  # the same kernel as attend_tree's
            assert torch.equal(out.view(own.shape), own)
        assert bool((buffer[:offset] == 7).all())
        assert bool((buffer[offset + own.numel():] == 7).all())
    assert not _lib.device_flags(DEV)
