"""Frame-attention calls with a tensor on another device than the context's are refused before the
library is called. No device: tensors that say where they are, and a library that counts calls."""
from __future__ import annotations

import types

import pytest
import torch

from jasnamacos_amd import frame_attention as fa
from jasnamacos_amd.deform_conv import INVALID_ARGUMENT, DeformConvError

BF16, I32, F32 = torch.bfloat16, torch.int32, torch.float32


class Placed(torch.Tensor):
    where = 0
    is_cuda = True

    def get_device(self):
        return self.where


def on(where, t):
    t = t.as_subclass(Placed)
    t.where = where
    return t


def t(*shape, dtype=BF16):
    return on(0, torch.zeros(*shape, dtype=dtype))


class Library:
    """Every function succeeds, every size is 0."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def call(*a):
            self.calls += name.endswith("_dev")
            return 0
        return call


def calls(ctx):
    """name: (call, its arguments)."""
    rotary, attention, norm = fa.Rotary(ctx, 64, (16, 8, 8)), fa.FrameAttention(ctx, 4, 2, 64), fa.GatedNorm(ctx, 64, 4)
    q, k, lse = t(8, 4, 64), t(8, 2, 64), t(8, 4, dtype=F32)
    pages, table, lens = t(2, 16, 2, 64), t(1, 2, dtype=I32), t(1, dtype=I32)
    cu, positions, freq = t(2, dtype=I32), t(8, 3, dtype=I32), t(32, dtype=F32)
    row, w, gate, sums, rstd = t(8, 64), t(64), t(2, 64), t(64, dtype=F32), t(8, 2, dtype=F32)
    return {
        "rotary": (rotary.run_dev, {"x": q, "positions": positions, "freq": freq, "out": q}),
        "append": (fa.CacheAppend(ctx).run_dev, {"k": k, "v": k, "k_pages": pages, "v_pages": pages, "table": table, "cu_q": cu,
                                                 "kv_lens": lens, "rotary": rotary, "positions": positions, "freq": freq,
                                                 "q": q, "q_out": q}),
        "forward": (attention.forward_dev, {"q": q, "k": k, "v": k, "out": q, "lse": lse, "cu_q": cu, "cu_kv": cu}),
        "backward": (attention.backward_dev, {"q": q, "k": k, "v": k, "out": q, "lse": lse, "dout": q, "dq": q, "dk": k, "dv": k,
                                              "cu_q": cu, "cu_kv": cu}),
        "paged": (attention.paged_dev, {"q": q, "k_pages": pages, "v_pages": pages, "table": table, "cu_q": cu, "kv_lens": lens,
                                        "out": q, "lse": lse}),
        "norm": (norm.forward_dev, {"h": row, "x": row, "gate": gate, "w_post": w, "w_pre": w, "x_out": row, "y": row,
                                    "rstd": rstd}),
        "norm backward": (norm.backward_dev, {"h": row, "x_out": row, "gate": gate, "w_post": w, "w_pre": w, "rstd": rstd,
                                              "dx_out": row, "dy": row, "dh": row, "dx": row, "dgate": gate, "dw_post": sums,
                                              "dw_pre": sums}),
    }


@pytest.mark.parametrize("name", ["rotary", "append", "forward", "backward", "paged", "norm", "norm backward"])
def test_tensors_of_another_device(name):
    lib = Library()
    ctx = types.SimpleNamespace(ctx=None, device=0, _lib=lib, _check=lambda status: None)
    call, args = calls(ctx)[name]
    call(**args)
    assert lib.calls == 1
    for key, value in args.items():
        if not isinstance(value, torch.Tensor):
            continue
        for where in (1, -1):
            with pytest.raises(DeformConvError) as e:
                call(**{**args, key: on(where, value.clone())})
            assert e.value.status == INVALID_ARGUMENT and lib.calls == 1, key


def test_low_of_another_device():
    lib = Library()
    lib.dcn_gated_norm_low_bytes = lambda s: 1024
    ctx = types.SimpleNamespace(ctx=None, device=0, _lib=lib, _check=lambda status: None)
    call, args = calls(ctx)["norm"]
    call(**args, low=t(1024, dtype=torch.uint8))
    with pytest.raises(DeformConvError) as e:
        call(**args, low=on(1, torch.zeros(1024, dtype=torch.uint8)))
    assert e.value.status == INVALID_ARGUMENT and lib.calls == 1


def test_context_of_another_device():
    ctx = types.SimpleNamespace(ctx=None, device=1, _lib=Library(), _check=lambda status: None)
    call, args = calls(ctx)["norm"]
    with pytest.raises(DeformConvError, match="on device 0; the context is on 1"):
        call(**args)
