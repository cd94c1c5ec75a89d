"""Bounds of the sequences' lengths: however loose, the same plan and workspace as tight ones."""
from __future__ import annotations

import pytest

from jasnamacos_amd import _lib
from jasnamacos_amd import frame_attention as fa

MOST = 2**31 - 1


def workspace(which, dtype=1, q_heads=8, kv_heads=1, dim=64, frame=1, back=-1, ahead=0, sinks=0, max_q=2000, max_kv=300,
              q_tokens=2000, kv_tokens=300, sequences=1):
    s = fa._ATTENTION.pack(dtype, sequences, q_heads, kv_heads, dim, frame, back, ahead, sinks, max_q, max_kv, 1.0, q_tokens,
                           kv_tokens, *[0] * 16)
    return _lib.load().dcn_attention_workspace_bytes(s, which)


@pytest.mark.parametrize("window", [{}, {"back": 100, "sinks": 40}, {"back": MOST, "ahead": MOST, "frame": MOST},
                                    {"back": 0, "frame": MOST, "sinks": 1}])
def test_backward(window):
    """2,000 rows of 8 heads over three blocks of keys: split in parts, which the workspace holds."""
    tight = workspace(fa.PASS_BACKWARD, **window)
    assert tight > 2000 * 8 * 4
    assert workspace(fa.PASS_BACKWARD, max_kv=MOST, **window) == tight
    assert workspace(fa.PASS_BACKWARD, max_q=MOST, **window) == tight


@pytest.mark.parametrize("dtype", [1, 2])
def test_forward(dtype):
    few = dict(dtype=dtype, max_q=1, q_tokens=1, q_heads=8, kv_heads=8, kv_tokens=20000)
    tight = workspace(fa.PASS_FORWARD, **{**few, "max_kv": 20000})
    assert tight > 0 and workspace(fa.PASS_FORWARD, **{**few, "max_kv": MOST, "max_q": MOST}) == tight


def test_windows_past_the_rows():
    """A window longer than the queries is no window."""
    assert workspace(fa.PASS_BACKWARD, back=MOST, ahead=MOST, frame=65536) == workspace(fa.PASS_BACKWARD, ahead=-1)


@pytest.mark.parametrize("shape", [
    dict(sequences=64, q_heads=32, kv_heads=8, dim=128, back=100, sinks=2000, max_q=2000, max_kv=2000),
    dict(sequences=4, q_heads=8, kv_heads=8, back=16, sinks=4096, max_q=8192, max_kv=8192),
    dict(q_heads=8, kv_heads=8, back=16, sinks=4096, max_q=65536, max_kv=65536),
    dict(q_heads=2, kv_heads=1, frame=2**31 - 1, back=0, sinks=1, max_q=300, max_kv=300)])
def test_many_sinks(shape):
    """The parts of the sinks' gradients: four workgroups a CU of 2 x 128 FP32 rows at most."""
    tokens = shape.get("sequences", 1) * shape["max_q"]
    rows = (tokens * shape["q_heads"] + 3) // 4 * 4
    assert workspace(fa.PASS_BACKWARD, **shape, q_tokens=tokens, kv_tokens=tokens) <= 4 * (rows + 1024 * 2 * 128 * shape.get("dim", 64))


@pytest.mark.parametrize("keys,parts", [(8000, 31), (540, 2), (300, 1)])
def test_fp32_heads_in_parts(keys, parts):
    """One token, 8 heads of 64: a workgroup a CU, of eight waves with a tile of 32 keys each at least."""
    size = workspace(fa.PASS_FORWARD, dtype=2, q_heads=8, kv_heads=8, max_q=1, q_tokens=1, max_kv=keys, kv_tokens=keys)
    assert size == (8 * parts * (64 + 4) * 4 if parts > 1 else 0)
