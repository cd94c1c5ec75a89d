"""The microscaled cache in 64 bits, on the CPU: blocks of 32 channels share a power of two,
codes are e4m3 (8 bits) or e2m1 (4)."""
from __future__ import annotations

import torch

LARGEST = {8: 448.0, 4: 6.0}
# The largest magnitude that is written, by type: its code reads back as a finite value.
MOST = {(torch.float16, 8): 61440.0, (torch.float16, 4): 49152.0, (torch.bfloat16, 8): 1.875 * 2.0**127,
        (torch.bfloat16, 4): 1.5 * 2.0**127, (torch.float32, 8): 1.875 * 2.0**127, (torch.float32, 4): 1.5 * 2.0**127}
# Half a step of a code, relative (normal codes) and absolute (the smallest ones), in units of the block's power of two.
HALF = {8: (2.0**-4, 2.0**-10), 4: (2.0**-2, 2.0**-2)}


def code_values(bits):
    """What each code stands for, from its fields."""
    width, bias, fraction = (4, 7, 3) if bits == 8 else (2, 1, 1)
    values = []
    for code in range(1 << bits):
        e, f = (code >> fraction) & ((1 << width) - 1), code & ((1 << fraction) - 1)
        size = (1 + f / (1 << fraction)) * 2.0 ** (e - bias) if e else f / (1 << fraction) * 2.0 ** (1 - bias)
        if bits == 8 and code & 127 == 127:
            size = float("nan")
        values.append(-size if code >> (bits - 1) else size)
    return torch.tensor(values, dtype=torch.float64)


def nearest(x, bits):
    """The code of each value (magnitudes within the largest), ties to the even code."""
    values = code_values(bits)[: 1 << (bits - 1)]
    values = values[torch.isfinite(values)]
    size = x.abs().contiguous()
    above = torch.searchsorted(values, size).clamp(max=len(values) - 1)
    below = (above - 1).clamp(min=0)
    d_above, d_below = values[above] - size, size - values[below]
    index = torch.where((d_below < d_above) | ((d_below == d_above) & (below % 2 == 0)), below, above)
    return index + torch.signbit(x).long() * (1 << (bits - 1))


def quantise(x, bits, dtype):
    """(codes [...][dim], scale bytes [...][dim / 32]) of values, as a cache of tensors of `dtype` keeps them."""
    most = MOST[dtype, bits]
    blocks = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(blocks).all(-1)
    blocks = torch.where(bad[..., None], torch.zeros_like(blocks), blocks).clamp(-most, most)
    top = blocks.abs().amax(-1)
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for k in range(-126, 128):
        e[top > LARGEST[bits] * 2.0 ** (k - 1)] = k
    codes = nearest(blocks * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e.double())[..., None], bits)
    return codes.flatten(-2), torch.where(bad, 255, e + 127)


def pack(codes, bits):
    codes = codes.to(torch.uint8)
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def values(packed, scales, bits):
    """[...][dim] in 64 bits of bytes of codes and scales."""
    codes = packed.long() if bits == 8 else torch.stack([packed & 15, packed >> 4], -1).flatten(-2).long()
    factor = torch.where(scales == 255, float("nan"), torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127))
    return (code_values(bits)[codes].unflatten(-1, (-1, 32)) * factor[..., None]).flatten(-2)


def to_pages(x, table, page, pages, bits, dtype, fill=0x5A):
    """Buffers (codes, scales) of a cache that holds x[s] ([tokens][heads][dim]) of each sequence."""
    heads, dim = x[0].shape[1:]
    codes = torch.full((pages, heads, page, dim * bits // 8), fill, dtype=torch.uint8)
    scales = torch.full((pages, heads, page, dim // 32), fill, dtype=torch.uint8)
    for s, rows in enumerate(x):
        if not len(rows):
            continue
        c, e = quantise(rows, bits, dtype)
        at = torch.arange(len(rows))
        which = table[s][at // page].long()
        codes[which, :, at % page] = pack(c, bits)
        scales[which, :, at % page] = e.to(torch.uint8)
    return codes, scales


def from_pages(codes, scales, table, n, page, bits):
    """[n][heads][dim] in 64 bits of one sequence."""
    at = torch.arange(n)
    which = table[at // page].long()
    return values(codes[which, :, at % page], scales[which, :, at % page], bits)
