"""GatedNorm's rounded-off halves: a backward uses those of the forward that made its rstd, whatever
other forwards ran in between, and without them takes x_out as it was rounded."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

TYPES = {"f16": "float16", "bf16": "bfloat16"}


class Step:
    """One call's tensors of a norm of `channels` channels, a gate for each run of five tokens."""

    def __init__(self, op, h, x, rstd=None):
        import torch

        self.op, self.h, self.x = op, h, x
        g = torch.Generator().manual_seed(8)
        tokens, c = h.shape
        self.w = torch.randn(c, generator=g).to(h.dtype).cuda()
        self.gate = torch.randn(-(-tokens // 5), c, generator=g).to(h.dtype).cuda()
        self.dx_out, self.dy = (torch.randn(tokens, c, generator=g).to(h.dtype).cuda() for _ in range(2))
        self.x_out, self.y = torch.empty_like(x), torch.empty_like(x)
        self.rstd = torch.empty(tokens, 2, device="cuda") if rstd is None else rstd

    def forward(self, low=None):
        self.op.forward_dev(self.h, self.x, self.gate, self.w, self.w, self.x_out, self.y, self.rstd, low)
        return self

    def backward(self, low=None, op=None, rstd=None):
        import torch

        dh, dx, dgate = torch.empty_like(self.h), torch.empty_like(self.x), torch.empty_like(self.gate)
        dw = [torch.empty(self.h.shape[1], device="cuda") for _ in range(2)]
        (op or self.op).backward_dev(self.h, self.x_out, self.gate, self.w, self.w, self.rstd if rstd is None else rstd,
                                     self.dx_out, self.dy, dh, dx, dgate, *dw, low=low)
        torch.cuda.synchronize()
        return [t.cpu() for t in (dh, dx, dgate, *dw)]


def make(fa, gpu_ctx, name, tokens=50, channels=64):
    """(handle, h, x, what the backward gives with the halves, without them)."""
    import torch

    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(7)
    h, x = (torch.randn(tokens, channels, generator=g).to(dtype).cuda() for _ in range(2))
    new = lambda: fa.GatedNorm(gpu_ctx, channels, 5)  # noqa: E731
    low = torch.empty(new().low_bytes(x), dtype=torch.uint8, device="cuda")
    step = Step(new(), h, x).forward(low)
    return new(), h, x, step.backward(low), step.backward(op=new())


def same(a, b):
    import torch

    return all(torch.equal(i, j) for i, j in zip(a, b))


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("tokens,channels", [(50, 64), (16, 8), (33, 257), (1, 1032)])
def test_last_forward(fa, gpu_ctx, name, tokens, channels):
    """The handle's own halves serve its last forward's backward, rstd given as another view too."""
    print("case: last forward", name, tokens, channels, flush=True)
    op, h, x, whole, rounded = make(fa, gpu_ctx, name, tokens, channels)
    assert not same(whole, rounded)
    step = Step(op, h, x).forward()
    assert same(step.backward(), whole)
    assert same(step.backward(rstd=step.rstd.view(-1).view(-1, 2)), whole)
    assert same(step.backward(op=fa.GatedNorm(gpu_ctx, channels, 5)), rounded)


@pytest.mark.parametrize("name", TYPES)
def test_another_forward_of_the_same_statistics(fa, gpu_ctx, name):
    """(-h, -x) has the statistics of (h, x) to the bit."""
    import torch

    print("case: negated", name, flush=True)
    op, h, x, whole, rounded = make(fa, gpu_ctx, name)
    first, second = Step(op, h, x).forward(), Step(op, -h, -x).forward()
    torch.cuda.synchronize()
    assert torch.equal(first.rstd, second.rstd)
    assert same(first.backward(), rounded)
    low = torch.empty(op.low_bytes(x), dtype=torch.uint8, device="cuda")
    first = Step(op, h, x).forward(low)
    Step(op, -h, -x).forward()
    assert same(first.backward(low), whole)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("more", [100, 17])
def test_a_forward_of_another_length(fa, gpu_ctx, name, more):
    """Rows that two calls of different lengths share, through the handle and through the caller's low."""
    import torch

    print("case: another length", name, more, flush=True)
    op, h, x, whole, rounded = make(fa, gpu_ctx, name)
    g = torch.Generator().manual_seed(9)
    extra = [torch.randn(100, 64, generator=g).to(h.dtype).cuda() for _ in range(2)]
    for t, own in zip(extra, (h, x)):
        t[:50] = own
    other = [t[:more].contiguous() for t in extra]
    first = Step(op, h, x).forward()
    second = Step(op, *other)
    second.gate[:min(10, len(second.gate))] = first.gate[:min(10, len(second.gate))]
    second.forward()
    torch.cuda.synchronize()
    rows = min(50, more)
    assert torch.equal(first.rstd[:rows], second.rstd[:rows])
    assert same(first.backward(), rounded)
    low = torch.empty(op.low_bytes(extra[0]), dtype=torch.uint8, device="cuda")
    first.forward(low)
    second.forward(low)
    assert same(first.backward(low), whole)


@pytest.mark.parametrize("name", TYPES)
def test_rstd_of_a_forward_elsewhere(fa, gpu_ctx, name):
    """A forward that keeps its halves with the caller writes the rstd of an earlier one."""
    import torch

    print("case: rstd elsewhere", name, flush=True)
    op, h, x, whole, rounded = make(fa, gpu_ctx, name)
    low = torch.empty(op.low_bytes(x), dtype=torch.uint8, device="cuda")
    negated = Step(op, -h, -x).forward()
    step = Step(op, h, x, negated.rstd).forward(low)
    assert same(step.backward(), rounded) and same(step.backward(low), whole)
