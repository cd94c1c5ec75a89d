"""Frame-attention calls with a tensor that is missing or not on the device are refused before
anything is launched."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, I32, F32 = torch.bfloat16, torch.int32, torch.float32


def t(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def calls(ctx):
    """name: (call, its arguments, which of them may be missing)."""
    from jasnamacos_amd import frame_attention as fa

    rotary, attention, norm = fa.Rotary(ctx, 64, (16, 8, 8)), fa.FrameAttention(ctx, 4, 2, 64), fa.GatedNorm(ctx, 64, 4)
    q, k, lse = t(8, 4, 64), t(8, 2, 64), t(8, 4, dtype=F32)
    pages, table, lens = t(2, 16, 2, 64), t(1, 2, dtype=I32), t(1, dtype=I32)
    cu, positions, freq = torch.tensor([0, 8], dtype=I32, device="cuda"), t(8, 3, dtype=I32), t(32, dtype=F32)
    row, w, gate = t(8, 64), t(64), t(2, 64)
    sums, rstd = t(64, dtype=F32), t(8, 2, dtype=F32)
    low = torch.zeros(norm.low_bytes(row), dtype=torch.uint8, device="cuda")
    return {
        "rotary": (rotary.run_dev, {"x": q, "positions": positions, "freq": freq, "out": t(8, 4, 64)}, ()),
        "append": (fa.CacheAppend(ctx).run_dev, {"k": k, "v": k, "k_pages": pages, "v_pages": t(2, 16, 2, 64), "table": table, "cu_q": cu,
                                      "kv_lens": lens, "rotary": rotary, "positions": positions, "freq": freq, "q": q,
                                      "q_out": t(8, 4, 64)}, ("q", "rotary")),
        "forward": (attention.forward_dev, {"q": q, "k": k, "v": k, "out": t(8, 4, 64), "lse": lse, "cu_q": cu, "cu_kv": cu},
                    ("lse", "cu_q", "cu_kv")),
        "backward": (attention.backward_dev, {"q": q, "k": k, "v": k, "out": q, "lse": lse, "dout": q, "dq": t(8, 4, 64),
                                              "dk": t(8, 2, 64), "dv": t(8, 2, 64)}, ()),
        "paged": (attention.paged_dev, {"q": q, "k_pages": pages, "v_pages": pages, "table": table, "cu_q": cu, "kv_lens": lens,
                                        "out": t(8, 4, 64), "lse": lse}, ("lse", "cu_q")),
        "norm": (norm.forward_dev, {"h": row, "x": row, "gate": gate, "w_post": w, "w_pre": w, "x_out": t(8, 64), "y": t(8, 64),
                                    "rstd": rstd, "low": low}, ("gate", "w_post", "w_pre", "y", "rstd", "low")),
        "norm backward": (norm.backward_dev, {"h": row, "x_out": row, "gate": gate, "w_post": w, "w_pre": w, "rstd": rstd,
                                              "dx_out": row, "dy": row, "dh": t(8, 64), "dx": t(8, 64), "dgate": t(2, 64),
                                              "dw_post": sums, "dw_pre": t(64, dtype=F32), "low": low},
                          ("gate", "w_post", "w_pre", "dy", "dgate", "dw_post", "dw_pre", "low")),
    }


@pytest.mark.parametrize("name", ["rotary", "append", "forward", "backward", "paged", "norm", "norm backward"])
def test_missing_or_on_the_host(name, gpu_ctx):
    from jasnamacos_amd.deform_conv import DeformConvError

    call, args, optional = calls(gpu_ctx)[name]
    call(**args)
    for key, value in args.items():
        for bad in [None] * (key not in optional) + ([value.cpu()] if isinstance(value, torch.Tensor) else []):
            with pytest.raises(DeformConvError) as e:
                call(**{**args, key: bad})
            assert e.value.status != 0, key
    torch.cuda.synchronize()
