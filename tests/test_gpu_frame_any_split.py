"""FrameAttention of any type where rows are few and keys many: workgroups share a row's keys and
their parts are joined. Against the definition in 64 bits, bounds as in frame_attention_reference."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def check(got, lse, q, k, v, seen, dtype, group):
    import frame_attention_reference as ref

    for h in range(q.shape[1]):
        want = ref.attention(q[:, h], k[:, h // group], v[:, h // group], seen, 1 / math.sqrt(q.shape[2]), dtype)
        for key, t in (("out", got), ("lse", lse)):
            value, bound = want[key]
            mine = t[:, h].double()
            same = (mine == value) | ((mine - value).abs() <= bound)
            assert same.all(), f"{key} head {h}: {((mine - value).abs() / bound).nan_to_num(0).max()}"


# dtype, head_dim, q_heads, kv_heads, queries, keys, frame, back, sinks
@pytest.mark.parametrize("case", [
    ("f32", 64, 4, 2, 1, 3001, 1, -1, 0),
    ("f32", 128, 3, 1, 19, 2050, 7, 200, 2),
    ("f32", 200, 2, 2, 5, 1111, 1, -1, 0),
    ("bf16", 33, 8, 2, 3, 4099, 16, 120, 1),
    ("f16", 1, 1, 1, 2, 1500, 1, -1, 0),
], ids=lambda c: f"{c[0]}-{c[1]}-{c[4]}x{c[5]}")
def test_against_the_definition(case, gpu_ctx):
    import frame_attention_reference as ref
    from jasnamacos_amd import frame_attention as fa

    name, dim, q_heads, kv_heads, nq, nk, frame, back, sinks = case
    dtype = TYPES[name]
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(n, heads, dim, generator=g).to(dtype) for n, heads in ((nq, q_heads), (nk, kv_heads), (nk, kv_heads)))
    op = fa.FrameAttention(gpu_ctx, q_heads, kv_heads, dim, frame, back, 0, sinks)
    results = []
    for _ in range(2):
        out = torch.full_like(q, math.nan, device="cuda")
        lse = torch.full((nq, q_heads), math.nan, device="cuda")
        op.forward_dev(q.cuda(), k.cuda(), v.cuda(), out, lse)
        results.append((out.cpu(), lse.cpu()))
    assert op._workspace is not None  # there were parts
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    check(*results[0], q, k, v, ref.visible(nq, nk, frame, back, 0, sinks), dtype, q_heads // kv_heads)


@pytest.mark.parametrize("dim", [64, 129])
def test_paged_with_ragged_histories(dim, gpu_ctx):
    """Sequences of no, one, a few and many keys in one call: most of their parts are empty. Unused
    rows of pages hold NaN."""
    import frame_attention_reference as ref
    from jasnamacos_amd.frame_attention import FrameAttention

    dtype, q_heads, kv_heads, page, lens = torch.float32, 4, 2, 16, [0, 1, 70, 2501]
    g = torch.Generator().manual_seed(6)
    width = -(-max(lens) // page)
    table = torch.randperm(len(lens) * width, generator=g).view(len(lens), width).to(torch.int32)
    pages = [torch.full((len(lens) * width, page, kv_heads, dim), math.nan, dtype=dtype) for _ in range(2)]
    q = torch.randn(len(lens), q_heads, dim, generator=g).to(dtype)
    rows = []
    for s, n in enumerate(lens):
        rows.append([torch.randn(n, kv_heads, dim, generator=g).to(dtype) for _ in range(2)])
        at = torch.arange(n)
        for t, p in zip(rows[s], pages):
            p[table[s, at // page].long(), at % page] = t
    op = FrameAttention(gpu_ctx, q_heads, kv_heads, dim)
    out, lse = torch.full_like(q, math.nan, device="cuda"), torch.full((len(lens), q_heads), math.nan, device="cuda")
    op.paged_dev(q.cuda(), pages[0].cuda(), pages[1].cuda(), table.cuda(), None,
                 torch.tensor(lens, dtype=torch.int32, device="cuda"), out, lse)
    assert op._workspace is not None
    for s, n in enumerate(lens):
        check(out[s:s + 1].cpu(), lse[s:s + 1].cpu(), q[s:s + 1], *rows[s], ref.visible(1, n, 1, -1, 0, 0), dtype, 2)


def test_values_that_are_not_finite(gpu_ctx):
    """A NaN that the last row sees and the first does not, in the last part: that channel of the last
    row is NaN, all else as with a zero there."""
    from jasnamacos_amd.frame_attention import FrameAttention

    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(n, 1, 64, generator=g) for n in (2, 2000, 2000))
    op = FrameAttention(gpu_ctx, 1, 1, 64)
    outs = []
    for value in (0.0, math.nan):
        v[1999, 0, 5] = value
        out = torch.empty(2, 1, 64, device="cuda")
        op.forward_dev(q.cuda(), k.cuda(), v.cuda(), out)
        outs.append(out.cpu())
    assert op._workspace is not None
    assert torch.equal(outs[0][0], outs[1][0])
    assert outs[1][1, 0, 5].isnan() and torch.equal(outs[0][1, 0, 6:], outs[1][1, 0, 6:])


def test_captured(gpu_ctx):
    """A graph of a call with parts, replayed between other work, as the eager call."""
    from jasnamacos_amd.frame_attention import FrameAttention

    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(n, 2, 64, generator=g).cuda() for n in (1, 4000, 4000))
    op = FrameAttention(gpu_ctx, 2, 2, 64)
    want, out = torch.empty_like(q), torch.empty_like(q)
    op.forward_dev(q, k, v, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.forward_dev(q, k, v, out, stream=torch.cuda.current_stream())
    for _ in range(4):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        op.forward_dev(q, k, v, want)
        torch.cuda.synchronize()
