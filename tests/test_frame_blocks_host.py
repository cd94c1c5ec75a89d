"""The example's blocks without a device: which handles they use, what serving leaves out, and that
second derivatives are refused. The operators' calls are recorded, not run."""
from __future__ import annotations

import types

import pytest
import torch

from jasnamacos_amd import _lib
from jasnamacos_amd import frame_attention as fa
from jasnamacos_amd import frame_blocks as fb


@pytest.fixture
def blocks(monkeypatch):
    """(FrameBlocks, used handles, the current stream)."""
    used, stream = [], types.SimpleNamespace(cuda_stream=0)

    def current_stream(device=None):
        assert device == torch.device("cpu")  # the blocks' own, not the current device's
        return stream
    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    for kind, calls in ((fa.FrameAttention, ("forward_dev", "backward_dev", "paged_dev")), (fa.GatedNorm, ("forward_dev", "backward_dev"))):
        for call in calls:
            monkeypatch.setattr(kind, call, lambda self, *a, **kw: used.append(self))
    for kind in (fa.Rotary, fa.CacheAppend):
        monkeypatch.setattr(kind, "run_dev", lambda self, *a, **kw: None)
    ctx = types.SimpleNamespace(ctx=None, device=0, _lib=_lib.load())
    return fb.FrameBlocks(ctx, 48, 4, 2, 16, 2, 2, 3, 1, 1, torch.float32, device="cpu"), used, stream


def test_handles(blocks):
    net, used, stream = blocks

    def handles(call):
        used.clear()
        call()
        return {id(h) for h in used}

    x, style = torch.randn(18, 48, requires_grad=True), torch.randn(3, 48)
    frame = x.detach()[:6], style[:1]
    sets, kept = [], []
    for stream.cuda_stream in (0, 7):
        one = handles(lambda: net.clip(x, style))
        assert len(one) == 2
        y = net.clip(x, style)
        assert handles(lambda: y.sum().backward()) == one
        assert handles(lambda: net.clip(x, style)) == one  # kept, not made for each call
        sets.append(one)
    for _ in range(2):
        serving = net.stream(1, 4, 2)
        one = handles(lambda: serving.step(*frame))
        assert len(one) == 2 and handles(lambda: serving.step(*frame)) == one
        sets.append(one)
        kept.append(serving)  # alive: no other handle has its handles' ids
    assert len(set().union(*sets)) == sum(map(len, sets))


def test_second_derivatives_are_refused(blocks):
    """The operators have no gradient of their gradients: not a sum that leaves them out."""
    net, _, _ = blocks
    for w in net.parameters():
        w.requires_grad_()
    y = net.clip(torch.randn(18, 48), torch.randn(3, 48))
    grads = torch.autograd.grad(y.sum(), net.parameters(), create_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(g.square().sum() for g in grads if g is not None).backward()


def test_serving_keeps_nothing_for_a_backward(blocks, monkeypatch):
    """Norms write their statistics and rounded-off halves where gradients are on."""
    net, _, _ = blocks
    kept = []

    def forward_dev(self, h, x, gate, w_post, w_pre, x_out, y=None, rstd=None, low=None, stream=None):
        kept.append(rstd is not None)
    monkeypatch.setattr(fa.GatedNorm, "forward_dev", forward_dev)
    x, style = torch.randn(18, 48), torch.randn(3, 48)
    net.stream(1, 4, 2).step(x[:6], style[:1])
    with torch.no_grad():
        net.clip(x, style)
    assert kept == [False] * 6
    net.clip(x, style)
    assert kept[6:] == [True] * 3
