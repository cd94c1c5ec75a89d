"""What a frame-attention handle keeps between calls: memory that a captured graph may hold the
address of is never given back."""
from __future__ import annotations

import types
import weakref

import pytest
import torch

from jasnamacos_amd import _lib
from jasnamacos_amd import frame_attention as fa


@pytest.fixture
def ctx(monkeypatch):
    """No device: the handles' memory comes from the host."""
    monkeypatch.setattr(fa, "_fresh", lambda count, like: torch.empty(count, dtype=torch.uint8))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    return types.SimpleNamespace(ctx=None, device=0, _lib=_lib.load())


def test_workspaces_that_calls_outgrow(ctx):
    op, x = fa.FrameAttention(ctx, 4, 2, 64), torch.zeros(1)
    address, size = op._room("small", lambda: 1000, x)
    first = weakref.ref(op._workspace)
    assert size >= 1000
    op._room("large", lambda: 5000, x)
    assert first() is not None and first().data_ptr() == address
    assert op._room("small", lambda: 1000, x)[1] >= 5000


def test_halves_that_calls_outgrow(ctx):
    op = fa.GatedNorm(ctx, 64)
    small, large = (torch.zeros(n, 64, dtype=torch.bfloat16) for n in (10, 100))
    address = op._low_to_write(op._pack(small), None, small, torch.zeros(10, 2))
    first = weakref.ref(op._kept)
    op._low_to_write(op._pack(large), None, large, torch.zeros(100, 2))
    assert first() is not None and first().data_ptr() == address
    assert op._kept.numel() >= op.low_bytes(large)


def test_many_small_steps_keep_little(ctx):
    """Calls that grow by a little each: what is kept in all stays within four times the last one's need."""
    op, x, made = fa.FrameAttention(ctx, 4, 2, 64), torch.zeros(1), []
    for count in range(1000, 9000, 16):
        assert op._room(count, lambda: count, x)[1] >= count
        if not made or made[-1]() is not op._workspace:
            made.append(weakref.ref(op._workspace))
    assert all(w() is not None for w in made)
    assert sum(w().numel() for w in made) <= 4 * 9000
