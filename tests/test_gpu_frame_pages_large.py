"""Attention over pages with as many workgroups as a launch may have, and with more."""
from __future__ import annotations

import pytest
import torch

from jasnamacos_amd.deform_conv import DeformConvError
from test_gpu_frame_large import repeats

pytestmark = pytest.mark.gpu

SEQUENCES, PERIOD = 65535, 3600  # lengths and tables repeat


def one_token_each(fa, ctx, heads, bits, sequences):
    """A call's queries, cache and the rest, as run() takes them."""
    g = torch.Generator().manual_seed(1)
    if bits:
        cache = fa.MxPages.zeros(3, 8, heads, 64, bits)
        for t, low, high in zip(cache._buffers, (0, 0, 118, 118), (127, 127, 123, 123)):
            t.copy_(torch.randint(low, high, t.shape, generator=g))
    else:
        cache = tuple(torch.randn(3, 8, heads, 64, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(PERIOD, heads, 64, generator=g).half().cuda().repeat(-(-sequences // PERIOD), 1, 1)[:sequences]
    s = torch.arange(sequences, device="cuda") % PERIOD
    return q, cache, (s % 3).int()[:, None].contiguous(), (s % 9).int()


def run(fa, ctx, heads, q, cache, table, lens):
    out, lse = torch.full_like(q, float("nan")), torch.full(q.shape[:2], float("nan"), device="cuda")
    none, length = torch.empty(0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    fa.FrameAttention(ctx, heads, heads, 64).shared_dev(q, cache, none, length, table, None, lens, out, lse)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("bits", [0, 8])
def test_past_2_22_workgroups(gpu_ctx, bits):
    """65,535 sequences of 65 heads: 4,259,776 workgroups."""
    from jasnamacos_amd import frame_attention as fa

    print("case: 2^22 workgroups", bits, flush=True)
    small, large = (run(fa, gpu_ctx, 65, *one_token_each(fa, gpu_ctx, 65, bits, n)) for n in (PERIOD, SEQUENCES))
    assert not any(torch.isnan(t).any() for t in small) and small[0].abs().max() > 0.1
    for want, got in zip(small, large):
        assert repeats(got, want)


def test_past_2_24_workgroups(gpu_ctx):
    """65,535 sequences of 258 heads are refused before anything is launched."""
    from jasnamacos_amd import frame_attention as fa

    print("case: 2^24 workgroups", flush=True)
    q, cache, table, lens = one_token_each(fa, gpu_ctx, 258, 8, SEQUENCES)
    out, length = torch.full_like(q, 7.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(DeformConvError):
        fa.FrameAttention(gpu_ctx, 258, 258, 64).paged_mx_dev(q, cache, table, None, lens, out)
    torch.cuda.synchronize()
    assert (out == 7.0).all()
