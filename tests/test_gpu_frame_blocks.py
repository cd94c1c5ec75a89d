"""The frame-attention operators together: blocks trained on clips and served from a cache."""
import math

import pytest
import torch

import frame_attention_reference as ref

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# channels, q_heads, kv_heads, head_dim, layers, rows, columns, back, sinks
SMALL = (48, 4, 2, 16, 2, 2, 3, 1, 1)
WIDE = (96, 4, 2, 64, 2, 4, 4, 2, 1)


def tolerance(dtype, sizes):
    """Of the relative distance between whole tensors. FP32: a dot product of n terms is off by
    n + 6 roundings at most, ten of them a block, growing at most four times through softmax and
    norms. 16 bits: eight roundings of a block's tensors (qkv, turned, weights, out, back, gate,
    x_out, y), each off by u at most, which also outweigh the sums' FP32."""
    blocks = sizes[4] + 1
    if dtype is torch.float32:
        return 2.0**-24 * (sizes[0] + 6) * 10 * 4 * blocks
    return ref.U[dtype] * 8 * blocks


def make(name, sizes):
    from jasnamacos_amd.deform_conv import HipDeformConv
    from jasnamacos_amd.frame_blocks import FrameBlocks

    channels, q_heads, kv_heads, head_dim, layers, rows, columns, back, sinks = sizes
    blocks = FrameBlocks(HipDeformConv(0), channels, q_heads, kv_heads, head_dim, layers, rows, columns, back, sinks,
                         DTYPES[name])
    return blocks, rows * columns


def data(g, dtype, *shape):
    return torch.randn(*shape, generator=g).to(dtype)


def plain(blocks, params, x, style, clips, sizes):
    """The blocks' output in 64 bits on the CPU, one head of one clip after the other."""
    channels, q_heads, kv_heads, head_dim, layers, rows, columns, back, sinks = sizes
    from jasnamacos_amd.frame_blocks import frame_positions

    n = len(x) // clips
    tokens = rows * columns
    positions = frame_positions(0, n // tokens, rows, columns, "cpu").repeat(clips, 1)
    freq = blocks.freq.cpu()
    seen = ref.visible(n, n, tokens, back, 0, sinks)
    eps, scale = blocks.norm.eps, 1.0 / math.sqrt(layers)
    y = x / torch.sqrt((x * x).mean(1, keepdim=True) + eps) * params[0]
    for i in range(layers):
        qkv, to, gate, w_post, w_pre = params[1 + 5 * i:6 + 5 * i]
        heads = (y @ qkv).view(len(x), -1, head_dim)
        turned = ref.rotate(heads[:, :q_heads + kv_heads], positions, freq, blocks.rotary.pairs, False, False)
        outs = []
        for c in range(clips):
            run = slice(c * n, (c + 1) * n)
            one = []
            for h in range(q_heads):
                kh = h // (q_heads // kv_heads)
                s = turned[run, h] @ turned[run, q_heads + kh].T / math.sqrt(head_dim)
                p = torch.softmax(s.masked_fill(~seen, -math.inf), 1)
                one.append(p @ heads[run, q_heads + kv_heads + kh])
            outs.append(torch.cat(one, 1))
        x, y = ref.gated_norm(torch.cat(outs) @ to, x, style @ gate, w_post, w_pre, tokens, scale, eps)
    return y


def apart(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("name,sizes", [("f32", SMALL), ("f16", WIDE), ("bf16", WIDE)])
def test_clip_and_its_gradients(name, sizes):
    blocks, tokens = make(name, sizes)
    g, dtype, clips, frames = torch.Generator().manual_seed(5), DTYPES[name], 2, 5
    x, style = data(g, dtype, clips * frames * tokens, sizes[0]), data(g, dtype, clips * frames, sizes[0])
    dy = data(g, dtype, *x.shape)
    params = [x.cuda(), style.cuda()] + blocks.parameters()
    for p in params:
        p.requires_grad_()
    y = blocks.clip(params[0], params[1], clips)
    y.backward(dy.cuda())
    exact = [p.detach().double().cpu().requires_grad_() for p in params]
    want = plain(blocks, exact[2:], exact[0], exact[1], clips, sizes)
    want.backward(dy.double())
    limit = tolerance(dtype, sizes)
    assert apart(y.detach(), want.detach()) < limit
    for i, (p, e) in enumerate(zip(params, exact)):
        assert apart(p.grad, e.grad) < 2 * limit, f"gradient of parameter {i}"


@pytest.mark.gpu
@pytest.mark.parametrize("name,sizes,page", [("f32", SMALL, 2), ("f16", WIDE, 16), ("bf16", WIDE, 8)])
def test_stream_gives_what_the_clip_does(name, sizes, page):
    """Three streams whose frames reuse the pages of those that left the window; pages start as NaN."""
    blocks, tokens = make(name, sizes)
    g, dtype, streams, frames = torch.Generator().manual_seed(6), DTYPES[name], 3, 8
    x = data(g, dtype, streams, frames, tokens, sizes[0]).cuda()
    style = data(g, dtype, streams, frames, sizes[0]).cuda()
    with torch.no_grad():
        whole = blocks.clip(x.view(-1, sizes[0]), style.view(-1, sizes[0]), streams).view(x.shape)
    serving = blocks.stream(streams, frames, page)
    for pages in serving.pages:
        for t in pages:
            t.fill_(math.nan)
    for f in range(frames):
        got = serving.step(x[:, f].reshape(-1, sizes[0]), style[:, f].contiguous())
        assert apart(got.view(streams, tokens, -1), whole[:, f].double().cpu()) < 2 * tolerance(dtype, sizes), f"frame {f}"
    with pytest.raises(ValueError, match="had their 8 frames"):
        serving.step(x[:, 0].reshape(-1, sizes[0]), style[:, 0].contiguous())


@pytest.mark.gpu
def test_stream_refusals():
    blocks, _ = make("f32", SMALL)
    with pytest.raises(ValueError, match="do not divide"):
        blocks.stream(1, 4, 4)
    blocks.back = -1
    with pytest.raises(ValueError, match="window with an end"):
        blocks.stream(1, 4, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_command(dtype, capsys):
    from jasnamacos_amd import frame_blocks

    assert frame_blocks.main(["--dtype", dtype, "--frames", "6", "--rows", "4", "--columns", "4", "--steps", "2"]) == 0
    assert "6 frames streamed" in capsys.readouterr().out


def test_positions():
    from jasnamacos_amd.frame_blocks import frame_positions

    got = frame_positions(3, 2, 2, 3, "cpu")
    assert got.dtype is torch.int32
    assert got.tolist() == [[f, r, c] for f in (3, 4) for r in range(2) for c in range(3)]
