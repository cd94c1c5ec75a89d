"""The 64-bit form of the microscaled cache against what its definition says."""
from __future__ import annotations

import pytest
import torch

import frame_mx_reference as mx


def test_codes():
    assert torch.equal(mx.code_values(8)[:127], torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double())
    assert mx.code_values(4)[:8].tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rounding(bits, dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(200, 64, generator=g) * torch.exp2(torch.randint(-20, 10, (200, 1), generator=g))).to(dtype)
    x[0] = 0
    codes, scales = mx.quantise(x, bits, dtype)
    back = mx.values(mx.pack(codes, bits), scales, bits)
    step = torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)
    near, small = mx.HALF[bits]
    assert ((back - x.double()).abs() <= torch.maximum(near * x.double().abs(), small * step)).all()
    top = x.double().abs().unflatten(-1, (-1, 32)).amax(-1)
    low = scales > 0
    assert (top <= mx.LARGEST[bits] * torch.pow(2.0, scales.double() - 127)).all()
    assert (top[low] > mx.LARGEST[bits] * torch.pow(2.0, scales[low].double() - 128)).all()
    assert (scales[0] == 0).all() and (codes[0] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_e4m3_as_torch_rounds(bits):
    """Every quarter step between codes, ties among them."""
    values = mx.code_values(bits)[: 1 << (bits - 1)]
    values = values[torch.isfinite(values)]
    x = torch.cat([values[:-1] + (values[1:] - values[:-1]) * part for part in (0, 0.25, 0.5, 0.75)] + [values[-1:]])
    codes = mx.nearest(x, bits)
    if bits == 8:
        assert torch.equal(codes, x.float().to(torch.float8_e4m3fn).view(torch.uint8).long())
    else:
        halves = codes[2 * 7:3 * 7]
        assert halves.tolist() == [0, 2, 2, 4, 4, 6, 6]
    assert torch.equal(mx.nearest(-x[1:], bits), codes[1:] + (1 << (bits - 1)))


def test_what_is_not_finite():
    x = torch.zeros(3, 64)
    x[0, 3], x[1, 40], x[2, 0] = float("inf"), float("nan"), 65504.0
    codes, scales = mx.quantise(x, 8, torch.float16)
    assert scales.tolist() == [[255, 0], [0, 255], [135, 0]]
    back = mx.values(codes, scales, 8)
    assert torch.isnan(back[0, :32]).all() and (back[0, 32:] == 0).all() and back[2, 0] == 61440
