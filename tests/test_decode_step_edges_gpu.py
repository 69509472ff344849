"""Decoding-step operators where types run out: small softmax weights, scores that tie, sums that cancel.

Held against the 64-bit definitions and bounds of ``decode_oracle``.
"""

import ctypes as ct

import pytest
import torch

from camblas_b200 import _kernels, _native
from tests import decode_oracle as exact
from tests.helpers import error_text, pointer, raw
from tests.test_decode_step_gpu import gen, int4_case, integers, normal, paged  # noqa: F401

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("heads,depth", [(3, 64), (16, 128), (4, 256)])
@pytest.mark.parametrize("ahead", [9.0, 12.5, 17.0, 20.0])
def test_small_weights_beside_a_dominant_token(gen, kind, heads, depth, ahead):
    """A first token that takes the weight and has the value zero: the result is made of the others' weights,
    e^-ahead of it."""
    length = 1500
    keys, values, table, counts = paged(gen, (length,), 16, 1, depth, BF16)
    first = int(table[0, 0])
    keys *= 0.25
    keys[..., 0] = 0
    keys[first, 0] = 0
    keys[first, 0, 0, 0] = 8
    values += 1
    values[first, 0] = 0
    keys, values = keys.to(kind), values.to(kind)
    q = (0.25 * normal(gen, 1, heads, depth)).to(BF16)
    q[..., 0] = 8
    out = _kernels.paged_attention(q, keys, values, table, counts, scale=ahead / 64)
    want, bound = exact.attention(q, keys, values, table, counts, ahead / 64, 0, 0)
    assert exact.within(out, want, bound)
