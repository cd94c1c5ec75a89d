"""FrameAttention with max_q and max_kv far above the lengths: the same bits as with the lengths."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,dim", [("bfloat16", 64), ("float16", 128), ("float32", 64), ("float16", 136)])
@pytest.mark.parametrize("bounds", [(2**31 - 1, 2**31 - 1), (250, 2**31 - 1), (2**31 - 1, 400), (1000, 1000)])
def test_loose_bounds(name, dim, bounds, gpu_ctx):
    import torch

    from jasnamacos_amd.frame_attention import FrameAttention

    print("case: bounds", name, dim, bounds, flush=True)
    dtype, g = getattr(torch, name), torch.Generator().manual_seed(1)
    r = lambda rows, heads: torch.randn(rows, heads, dim, generator=g).to(dtype).cuda()  # noqa: E731
    q, k, v, dout = r(250, 8), r(400, 2), r(400, 2), r(250, 8)
    starts = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 30, 250], [0, 100, 400])]
    op = FrameAttention(gpu_ctx, 8, 2, dim, 7, 12, 0, 1)

    def step(max_q, max_kv):
        out, lse = torch.full_like(q, math.nan), torch.empty(250, 8, device="cuda")
        grads = [torch.full_like(t, math.nan) for t in (q, k, v)]
        kw = dict(cu_q=starts[0], cu_kv=starts[1], max_q=max_q, max_kv=max_kv)
        op.forward_dev(q, k, v, out, lse, **kw)
        op.backward_dev(q, k, v, out, lse, dout, *grads, **kw)
        torch.cuda.synchronize()
        return [out, lse, *grads]

    # The bounds that there can be at most: plans, and the order of sums with them, go by the rows.
    want = step(250, 400)
    for a, b in zip(step(*bounds), want):
        assert torch.equal(a, b)


def test_equal_runs_are_still_checked(gpu_ctx):
    import torch

    from jasnamacos_amd.deform_conv import INVALID_SHAPE, DeformConvError
    from jasnamacos_amd.frame_attention import FrameAttention

    op, q = FrameAttention(gpu_ctx, 2, 2, 64), torch.zeros(8, 2, 64, dtype=torch.bfloat16, device="cuda")
    lib, out = gpu_ctx._lib, torch.zeros_like(q)
    for max_q, max_kv in ((9, 8), (8, 9)):  # one sequence of more rows than there are
        s = op._pack(q, 1, max_q, max_kv, 8, 8, *[q.stride()] * 4)
        assert lib.dcn_attention_forward_dev(gpu_ctx.ctx, s, q.data_ptr(), q.data_ptr(), q.data_ptr(), None, None, out.data_ptr(),
                                             None, None, 0, None) == INVALID_SHAPE
    with pytest.raises(DeformConvError):
        op.forward_dev(q, q, q, out, max_q=4, max_kv=5)
