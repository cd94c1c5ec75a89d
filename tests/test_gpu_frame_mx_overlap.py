"""An append into a microscaled cache whose turned queries are written where its inputs lie: refused; between
their rows: as anywhere else."""
from __future__ import annotations

import pytest
import torch

from jasnamacos_amd.deform_conv import DeformConvError

pytestmark = pytest.mark.gpu

TOKENS, Q, KV, DIM = 37, 4, 2, 64


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


def append(fa, ctx, q, k, v, q_out):
    cache = fa.MxPages.zeros(3, 16, KV, DIM)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rotary = fa.Rotary(ctx, DIM, (16, 8, 8))
    positions = (torch.arange(3 * TOKENS, dtype=torch.int32) % 29).view(TOKENS, 3).cuda()
    fa.CacheAppend(ctx).run_mx_dev(k, v, cache, i32(2, 0, 1)[None], i32(0, TOKENS), i32(TOKENS), rotary, positions, rotary.frequencies(), q, q_out)
    torch.cuda.synchronize()
    return cache


def inputs(heads):
    whole = torch.randn(TOKENS, heads, DIM, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    return whole, whole[:, :Q], whole[:, Q:Q + KV], whole[:, Q + KV:Q + 2 * KV]


@pytest.mark.parametrize("where", ["behind", "in front", "heads first"])
def test_between_the_rows(fa, gpu_ctx, where):
    print("case: between the rows", where, flush=True)
    whole, q, k, v = inputs(2 * Q + 2 * KV)
    if where == "in front":
        whole = torch.cat([torch.zeros_like(q), q, k, v], 1)
        q, k, v, q_out = whole[:, Q:2 * Q], whole[:, 2 * Q:2 * Q + KV], whole[:, 2 * Q + KV:], whole[:, :Q]
    elif where == "heads first":
        whole = whole.transpose(0, 1).contiguous()
        q, k, v, q_out = (t.transpose(0, 1) for t in whole.split((Q, KV, KV, Q)))
    else:
        q_out = whole[:, Q + 2 * KV:]
    want, before = torch.empty(TOKENS, Q, DIM, dtype=q.dtype, device="cuda"), [t.clone() for t in (q, k, v)]
    caches = [append(fa, gpu_ctx, q, k, v, to) for to in (want, q_out)]
    assert torch.equal(q_out, want) and all(torch.equal(a, b) for a, b in zip((q, k, v), before))
    assert all(torch.equal(a, b) for a, b in zip(caches[0]._buffers, caches[1]._buffers))


@pytest.mark.parametrize("first", [1, Q - 1, Q, Q + KV, Q + 2 * KV - 1])
def test_on_the_inputs(fa, gpu_ctx, first):
    print("case: on the inputs", first, flush=True)
    whole, q, k, v = inputs(2 * Q + 2 * KV)
    before = whole.clone()
    for q_out in (whole[:, first:first + Q], whole.view(-1, DIM)[first:first + TOKENS * Q].view(TOKENS, Q, DIM)):
        with pytest.raises(DeformConvError, match="q_out lies on"):
            append(fa, gpu_ctx, q, k, v, q_out)
        torch.cuda.synchronize()
        assert torch.equal(whole, before)
