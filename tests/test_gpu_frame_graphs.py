"""A captured graph of frame-attention calls goes on giving the same results after its handles
have grown, and writes nowhere else."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def replayed(step, results, grow):
    """Captures step() after one call of it, lets grow() outgrow the workspaces, fills new memory
    with a pattern, and replays: the results stay and the pattern is untouched."""
    import torch

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(side)
    side.synchronize()
    want = [t.clone() for t in results]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream())
    for _ in range(3):
        grow()
        torch.cuda.synchronize()
        pattern = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in (512, 4096, 40000, 200000, 1 << 20) for _ in range(8)]
        for t in results:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip(results, want):
            assert torch.equal(t, w)
        assert all((t == 77).all() for t in pattern)


def test_paged(gpu_ctx):
    import torch

    from jasnamacos_amd import frame_attention as fa

    print("case: graph of a paged call", flush=True)
    g = torch.Generator().manual_seed(1)

    def call(streams, keys):
        width = -(-keys // 64)
        pages = [torch.randn(streams * width, 64, 8, 64, generator=g).bfloat16().cuda() for _ in range(2)]
        table = torch.arange(streams * width, dtype=torch.int32, device="cuda").view(streams, width)
        lens = torch.full((streams,), keys, dtype=torch.int32, device="cuda")
        q = torch.randn(streams, 8, 64, generator=g).bfloat16().cuda()
        out = torch.empty_like(q)
        return out, lambda stream=None: op.paged_dev(q, *pages, table, None, lens, out, max_kv=keys, stream=stream)

    op = fa.FrameAttention(gpu_ctx, 8, 8, 64)
    out, small = call(1, 4096)
    large = [call(n, keys)[1] for n, keys in ((2, 4096), (4, 6000), (8, 8000))]
    calls = iter(large)
    replayed(small, [out], lambda: next(calls)())


def test_step_and_norm(gpu_ctx):
    """A training step's attention and norm, whose halves the handle keeps."""
    import torch

    from jasnamacos_amd import frame_attention as fa

    print("case: graph of a training step", flush=True)
    attention, norm = fa.FrameAttention(gpu_ctx, 4, 2, 64, back=40, sinks=1), fa.GatedNorm(gpu_ctx, 256, 10)
    g = torch.Generator().manual_seed(2)

    def call(tokens):
        r = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()  # noqa: E731
        q, k, v, dout = r(tokens, 4, 64), r(tokens, 2, 64), r(tokens, 2, 64), r(tokens, 4, 64)
        out, lse = torch.empty_like(q), torch.empty(tokens, 4, device="cuda")
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        x, dx_out, dy = r(tokens, 256), r(tokens, 256), r(tokens, 256)
        x_out, y, dh, dx = (torch.empty_like(x) for _ in range(4))
        rstd, dw = torch.empty(tokens, 2, device="cuda"), torch.empty(256, device="cuda")

        def step(stream=None):
            attention.forward_dev(q, k, v, out, lse, stream=stream)
            attention.backward_dev(q, k, v, out, lse, dout, dq, dk, dv, stream=stream)
            norm.forward_dev(out.flatten(1), x, None, None, None, x_out, y, rstd, stream=stream)
            norm.backward_dev(out.flatten(1), x_out, None, None, None, rstd, dx_out, dy, dh, dx, dw_pre=dw, stream=stream)
        return [out, dq, dk, dv, x_out, y, dh, dx, dw], step

    results, small = call(100)
    calls = iter([call(tokens)[1] for tokens in (200, 600, 2000)])
    replayed(small, results, lambda: next(calls)())
