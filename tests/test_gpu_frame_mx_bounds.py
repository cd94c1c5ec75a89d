"""Lengths that a table does not hold, over microscaled pages and behind a prefix: what lies past the table's width is
not written, not read, and not seen; lengths below zero are none."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, WIDTH, HEADS, DIM, PAGES = 16, 3, 2, 64, 9
NEW = [5, 7, 4, 6, 3]
LENS = [PAGE * WIDTH + 2, PAGE * WIDTH, PAGE * WIDTH + 40, -3, 2]  # past the width in part, up to it, wholly past it, below zero, fewer than are new


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts():
    cu = [0]
    for n in NEW:
        cu.append(cu[-1] + n)
    return cu


def tables():
    order = torch.randperm(PAGES, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    return torch.stack([order[:3], order[3:6], order[:3], order[6:], order[6:]])  # the third and the fourth write nothing


@pytest.mark.parametrize("bits", [8, 4])
def test_append_and_read(fa, gpu_ctx, bits):
    import frame_mx_reference as mx

    print("case: past the table", bits, flush=True)
    g, cu, table = torch.Generator().manual_seed(1), starts(), tables()
    k, v = (torch.randn(cu[-1], HEADS, DIM, generator=g).bfloat16() for _ in range(2))
    cache = fa.MxPages.zeros(PAGES, PAGE, HEADS, DIM, bits)
    for t in cache._buffers:
        t.fill_(0x5A)
    want = [t.cpu().clone() for t in cache._buffers]
    out = [torch.full(k.shape, 7.0, dtype=k.dtype, device="cuda") for _ in range(2)]
    back = [t.cpu().clone() for t in out]
    fa.CacheAppend(gpu_ctx).run_mx_dev(k.cuda(), v.cuda(), cache, table.cuda(), i32(*cu), i32(*LENS))
    fa.CacheRead(gpu_ctx).run_dev(cache, table.cuda(), i32(*cu), i32(*LENS), *out)
    torch.cuda.synchronize()
    for s, n in enumerate(LENS):
        for row in range(cu[s], cu[s + 1]):
            at = n - (cu[s + 1] - row)
            if 0 <= at < PAGE * WIDTH:
                page = int(table[s, at // PAGE])
                for part, x in enumerate((k, v)):
                    codes, scales = mx.quantise(x[row], bits, x.dtype)
                    want[part][page, :, at % PAGE], want[2 + part][page, :, at % PAGE] = mx.pack(codes, bits), scales.to(torch.uint8)
                    back[part][row] = mx.values(mx.pack(codes, bits), scales, bits).to(x.dtype)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(cache._buffers, want))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(out, back))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("prefix", [0, 20, 9000])
def test_attention(fa, gpu_ctx, prefix, bits, dtype):
    """As the same call with lengths that the table holds. A long prefix is read once for all of the
    sequences in 16 bits."""
    print("case: past the table", prefix, bits, dtype, flush=True)
    g, cu, dtype = torch.Generator().manual_seed(2), starts(), getattr(torch, dtype)
    heads = 8 if prefix > 1000 else HEADS
    pages = PAGES + -(-prefix // PAGE)
    if bits:
        cache = fa.MxPages.zeros(pages, PAGE, heads, DIM, bits)
        for t, low, high in zip(cache._buffers, (0, 0, 118, 118), (127, 127, 123, 123)):
            t.copy_(torch.randint(low, high, t.shape, generator=g))
    else:
        cache = tuple(torch.randn(pages, PAGE, heads, DIM, generator=g).to(dtype).cuda() for _ in range(2))
    copies = 12 if prefix > 1000 else 1
    new, lens, table = NEW * copies, LENS * copies, tables().repeat(copies, 1).cuda()
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], 2 * heads, DIM, generator=g).to(dtype).cuda()
    first = torch.arange(PAGES, pages, dtype=torch.int32, device="cuda")
    op, got = fa.FrameAttention(gpu_ctx, 2 * heads, heads, DIM), []
    for lengths in (lens, [min(max(n, 0), PAGE * WIDTH) for n in lens]):
        out, lse = torch.full_like(q, float("nan")), torch.full(q.shape[:2], float("nan"), device="cuda")
        op.shared_dev(q, cache, first, i32(prefix), table, i32(*cu), i32(*lengths), out, lse, max_q=max(new))
        torch.cuda.synchronize()
        got.append((out, lse))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert torch.isfinite(got[0][0]).all() and not torch.isnan(got[0][1]).any()
