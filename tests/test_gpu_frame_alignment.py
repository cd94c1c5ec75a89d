"""Pointers that are not aligned to their type are refused at the C entries, optional ones too."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_optional_pointers(dtype, gpu_ctx):
    import torch

    from jasnamacos_amd import frame_attention as fa
    from jasnamacos_amd.deform_conv import INVALID_ARGUMENT

    print("case: alignment", dtype, flush=True)
    lib, kind = gpu_ctx._lib, getattr(torch, dtype)
    room = {}

    def z(name, *shape, dtype=kind):
        room[name] = torch.zeros(*shape, dtype=dtype, device="cuda")
        return room[name].data_ptr()

    f32, i32 = torch.float32, torch.int32
    q, k, out = z("q", 8, 4, 64), z("k", 8, 2, 64), z("out", 8, 4, 64)
    dq, dk, dv = z("dq", 8, 4, 64), z("dk", 8, 2, 64), z("dv", 8, 2, 64)
    lse, cu, lens = z("lse", 9, 4, dtype=f32), z("cu", 3, dtype=i32), z("lens", 2, dtype=i32)
    table = z("table", 1, 2, dtype=i32)
    op = fa.FrameAttention(gpu_ctx, 4, 2, 64)
    wide, narrow = (256, 64), (128, 64)
    shape = op._pack(room["q"], 1, 8, 8, 8, 8, wide, narrow, narrow, wide, wide, wide, narrow, narrow)
    size = lib.dcn_attention_workspace_bytes(shape, fa.PASS_BACKWARD)
    work = z("work", size // 4 + 1, dtype=f32)
    pages = torch.zeros(2, 16, 2, 64, dtype=kind, device="cuda")
    cache = fa._cache(pages, pages, room["table"], 0)
    norm = fa.GatedNorm(gpu_ctx, 64, 4)
    rows = [z(n, 9, 64) for n in ("h", "x_out", "y", "dx_out", "dy", "dh", "dx", "gate", "dgate")]
    h, x_out, y, dx_out, dy, dh, dx, gate, dgate = rows
    w, rstd, dw1, dw2 = z("w", 65), z("rstd", 9, 2, dtype=f32), z("dw1", 65, dtype=f32), z("dw2", 65, dtype=f32)
    room["h"] = room["h"][:8]
    ns = norm._pack(room["h"])
    nsize = lib.dcn_gated_norm_workspace_bytes(ns)
    nwork = z("nwork", nsize // 4 + 1, dtype=f32)
    c = gpu_ctx.ctx
    entries = {  # call, arguments, those that may be null, their alignment
        "forward": (lib.dcn_attention_forward_dev, [c, shape, q, k, k, cu, cu, out, lse, work, size, None], {"cu_q": 5, "cu_kv": 6, "lse": 8}),
        "paged": (lib.dcn_attention_paged_dev, [c, shape, cache, q, pages.data_ptr(), pages.data_ptr(), cu, lens, table, out, lse, work,
                                                size, None], {"cu_q": 6, "lse": 10}),
        "backward": (lib.dcn_attention_backward_dev, [c, shape, q, k, k, out, lse, q, cu, cu, dq, dk, dv, work, size, None],
                     {"cu_q": 8, "cu_kv": 9}),
        "norm": (lib.dcn_gated_norm_forward_dev, [c, ns, h, x_out, gate, w, w, x_out, y, rstd, None, None],
                 {"gate": 4, "w_post": 5, "w_pre": 6, "y": 8, "rstd": 9}),
        "norm backward": (lib.dcn_gated_norm_backward_dev, [c, ns, h, x_out, gate, w, w, rstd, None, dx_out, dy, dh, dx, dgate, dw1, dw2,
                                                            nwork, nsize, None],
                          {"gate": 4, "w_post": 5, "w_pre": 6, "dy": 10, "dgate": 13, "dw_post": 14, "dw_pre": 15}),
    }
    for name, (call, args, optional) in entries.items():
        assert call(*args) == 0, (name, gpu_ctx.last_error)
        for key, at in optional.items():
            bad = list(args)
            bad[at] += 1
            assert call(*bad) == INVALID_ARGUMENT, (name, key)
            assert gpu_ctx.last_error == f"{key} is not aligned to its type"
    torch.cuda.synchronize()
