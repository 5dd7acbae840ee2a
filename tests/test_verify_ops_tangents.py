"""Inputs that carry a derivative are refused, in both directions of differentiation (the
check of the arguments runs on the host: no GPU needed)."""

import pytest
import torch
from torch.autograd import forward_ad

from hisparse_b200 import _lib


def test_forward_mode_tangents_are_refused():
    x = torch.randn(2, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for tensors in ((dual,), (x, None, dual), (x, x, dual * 2)):
            with pytest.raises(ValueError, match="no derivative"):
                _lib.one_device(*tensors)
            with torch.no_grad():  # has no effect on forward-mode differentiation
                with pytest.raises(ValueError, match="no derivative"):
                    _lib.one_device(*tensors)
        with torch.inference_mode():  # tangents are not followed here
            with pytest.raises(ValueError, match="CUDA"):
                _lib.one_device(dual)
        primal = forward_ad.unpack_dual(dual).primal
        with pytest.raises(ValueError, match="CUDA"):  # past the check
            _lib.one_device(x, primal)
    with pytest.raises(ValueError, match="CUDA"):
        _lib.one_device(x)


def test_reverse_mode_is_refused_as_before():
    x = torch.randn(2, 8, requires_grad=True)
    with pytest.raises(ValueError, match="no backward"):
        _lib.one_device(x.detach(), x)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        _lib.one_device(x)
