"""What the command of the frame blocks takes for a difference by roundings alone."""
from __future__ import annotations

import math

import pytest

from jasnamacos_amd.frame_blocks import _holds

TYPES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layers", [1, 2, 3, 24])
def test_what_is_wrong_does_not_pass(layers, dtype, bits):
    assert _holds(0.0, 0.0, layers, dtype, bits)
    for bad in (1.0, math.sqrt(2.0), math.inf, math.nan):  # zeros, other numbers of the same size, what is not finite
        assert not _holds(bad, 0.0, layers, dtype, bits)
        assert not _holds(0.0, bad, layers, dtype, bits)
        assert not _holds(bad, bad, layers, dtype, bits)


@pytest.mark.parametrize("dtype", TYPES)
def test_limits(dtype):
    """Of two blocks: codes of fewer bits allow a stream more, a continuation no more than BF16's roundings."""
    u = {"f16": 2.0**-8, "bf16": 2.0**-5, "f32": 2.0**-18}[dtype]
    for bits, codes in ((0, 0.0), (8, 0.072), (4, 0.289)):
        assert _holds(0.9 * (2 * u + codes), 0.0, 2, dtype, bits) and not _holds(1.1 * (2 * u + codes), 0.0, 2, dtype, bits)
        fork = 4 * (max(u, 2.0**-5) if bits else u)
        assert _holds(0.0, 0.9 * fork, 2, dtype, bits) and not _holds(0.0, 1.1 * fork, 2, dtype, bits)
