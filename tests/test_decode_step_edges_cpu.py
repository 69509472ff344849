"""Refusals of the decoding-step operators that need no GPU."""

import pytest
import torch

from camblas_b200 import _kernels
from tests.test_decode_step_cpu import bf16


def test_tangents_are_refused_like_gradients():
    """A dual tensor does not have requires_grad set; its tangent would be lost silently."""
    from torch.autograd import forward_ad

    value = bf16(2, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(value, torch.ones_like(value))
        with pytest.raises(ValueError, match="gradient"):
            _kernels._refuse_gradient(value, None, dual)
        with pytest.raises(ValueError, match="gradient"):
            _kernels.route_experts(dual, 2)
        with pytest.raises(ValueError, match="gradient"):
            _kernels.qk_norm_rope(dual.view(1, 2, 8), value.view(1, 2, 8), None, None, 0.0,
                                  torch.zeros(1, dtype=torch.int64), torch.zeros(1, 8))
        _kernels._refuse_gradient(value, None)
        with torch.no_grad():  # tangents go on under it
            with pytest.raises(ValueError, match="gradient"):
                _kernels._refuse_gradient(dual)
    _kernels._refuse_gradient(value, None)
