"""Frame attention: sizes and factors that the C structs' types do not hold are refused with the
package's own error."""
from __future__ import annotations

import types

import pytest
import torch

from jasnamacos_amd import _lib
from jasnamacos_amd import frame_attention as fa
from jasnamacos_amd.deform_conv import INVALID_SHAPE, DeformConvError


@pytest.fixture
def ctx():
    return types.SimpleNamespace(ctx=None, _lib=_lib.load())


def refused(call):
    with pytest.raises(DeformConvError) as e:
        call()
    assert e.value.status == INVALID_SHAPE


def test_rotary_sizes(ctx):
    refused(lambda: fa.Rotary(ctx, 2**31, (1, 1, 1)))
    refused(lambda: fa.Rotary(ctx, 64, (2**31, 0, 0)))


@pytest.mark.parametrize("factor", [float("inf"), float("nan")])
def test_factors_in_c(factor):
    """The C layer by itself: no workspace for what it refuses."""
    lib, zeros = _lib.load(), [0] * 16

    def attention(scale):
        s = fa._ATTENTION.pack(1, 1, 1, 1, 64, 1, -1, 0, 0, 8, 8, scale, 8, 8, *zeros)
        return lib.dcn_attention_workspace_bytes(s, fa.PASS_BACKWARD)

    def low(residual_scale, eps):
        return lib.dcn_gated_norm_low_bytes(fa._NORM.pack(0, 64, 2, 1, residual_scale, eps))
    assert attention(1.0) > 0 and attention(factor) == 0
    assert low(1.0, 0.0) > 0 and low(factor, 0.0) == 0 and low(1.0, factor) == 0


@pytest.mark.parametrize("factors", [{"residual_scale": 1e39}, {"eps": 1e39}, {"gate_tokens": 2**63}])
def test_norm_factors(ctx, factors):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    refused(lambda: fa.GatedNorm(ctx, 64, **{"gate_tokens": 1, **factors}).low_bytes(x))


@pytest.mark.parametrize("window", [{"frame_tokens": 2**31}, {"back": 2**31}, {"ahead": 2**31}, {"sinks": 2**31},
                                    {"scale": 1e39}])
def test_attention_windows(ctx, window):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    refused(lambda: fa.FrameAttention(ctx, 4, 2, 64, **window)._pack(q, 1, 2, 2, 2, 2))


def test_attention_lengths(ctx):
    """As a table so wide gives them: width x page_tokens past 2^31."""
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    refused(lambda: fa.FrameAttention(ctx, 4, 2, 64)._pack(q, 1, 2, 2**31, 2, 2))
