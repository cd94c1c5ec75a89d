"""Blocks over the tokens of a clip's frames, as an example of the frame-attention operators
used together: trained on whole clips, served frame by frame from a paged cache.

A block projects its input to queries, keys and values in one product, turns queries and keys
by their place in time, height and width (Rotary), lets every token see the frames before it
(FrameAttention), projects back, and adds the result to the residual stream under a gate for
each frame (GatedNorm, which also makes the next block's input). Serving appends each new
frame's keys and values to the pages (CacheAppend) and reads them there; the pages of frames
that have left the window take the newer ones, so a stream has a cache of sinks + back + 1
frames however many it is made for. No counterpart in the reference.

    python -m jasnamacos_amd.frame_blocks [--dtype bf16] [--frames 12] [--rows 16 --columns 16]

trains a few steps on a synthetic clip, then streams it and compares the two."""
from __future__ import annotations

import argparse
import math
import sys
import time

import torch
from torch.autograd.function import once_differentiable

from .deform_conv import HipDeformConv
from .frame_attention import CacheAppend, FrameAttention, GatedNorm, Rotary


def frame_positions(first: int, frames: int, rows: int, columns: int, device="cuda"):
    """[frames * rows * columns][3] int32: time, height and width of each token."""
    axes = (torch.arange(first, first + frames), torch.arange(rows), torch.arange(columns))
    grid = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1)
    return grid.reshape(-1, 3).to(torch.int32).to(device)


class _Attend(torch.autograd.Function):
    """qkv ([tokens][q, k and v heads]) -> the attention's output ([tokens][q heads])."""

    @staticmethod
    def forward(ctx, qkv, blocks, positions, longest):
        q, k, v = blocks.heads(qkv)
        turned = torch.empty(len(qkv), q.shape[1] + k.shape[1], q.shape[2], dtype=qkv.dtype, device=qkv.device)
        tq, tk = turned.split((q.shape[1], k.shape[1]), 1)
        out = torch.empty_like(tq, memory_format=torch.contiguous_format)
        lse = torch.empty(len(qkv), q.shape[1], dtype=torch.float32, device=qkv.device)
        stream = torch.cuda.current_stream(qkv.device)
        blocks.rotary.run_dev(q, positions, blocks.freq, tq, stream=stream)
        blocks.rotary.run_dev(k, positions, blocks.freq, tk, stream=stream)
        blocks.attention.forward_dev(tq, tk, v, out, lse, max_q=longest, max_kv=longest, stream=stream)
        ctx.save_for_backward(qkv, turned, out, lse, positions)
        ctx.blocks, ctx.longest = blocks, longest
        return out.flatten(1)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, turned, out, lse, positions = ctx.saved_tensors
        blocks, stream = ctx.blocks, torch.cuda.current_stream(qkv.device)
        _, _, v = blocks.heads(qkv)
        dqkv, dturned = torch.empty_like(qkv), torch.empty_like(turned)
        dq, dk, dv = blocks.heads(dqkv)
        tq, tk = turned.split((dq.shape[1], dk.shape[1]), 1)
        dtq, dtk = dturned.split((dq.shape[1], dk.shape[1]), 1)
        blocks.attention.backward_dev(tq, tk, v, out, lse, dout.contiguous().view_as(out), dtq, dtk, dv,
                                      max_q=ctx.longest, max_kv=ctx.longest, stream=stream)
        blocks.rotary.run_dev(dtq, positions, blocks.freq, dq, inverse=True, stream=stream)
        blocks.rotary.run_dev(dtk, positions, blocks.freq, dk, inverse=True, stream=stream)
        return dqkv, None, None, None


class _Norm(torch.autograd.Function):
    """(h, x, a gate for each frame, w_post, w_pre) -> (x_out, y)."""

    @staticmethod
    def forward(ctx, h, x, gate, w_post, w_pre, norm):
        x_out, y = torch.empty_like(x), torch.empty_like(x)
        rstd = torch.empty(len(x), 2, dtype=torch.float32, device=x.device)
        low = torch.empty(norm.low_bytes(x), dtype=torch.uint8, device=x.device)
        norm.forward_dev(h, x, gate, w_post, w_pre, x_out, y, rstd, low, stream=torch.cuda.current_stream(x.device))
        ctx.save_for_backward(h, x_out, gate, w_post, w_pre, rstd, low)
        ctx.norm = norm
        return x_out, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_out, dy):
        h, x_out, gate, w_post, w_pre, rstd, low = ctx.saved_tensors
        dh, dx, dgate = torch.empty_like(h), torch.empty_like(h), torch.empty_like(gate)
        dw_post = torch.empty(len(w_post), dtype=torch.float32, device=h.device)
        dw_pre = torch.empty_like(dw_post)
        ctx.norm.backward_dev(h, x_out, gate, w_post, w_pre, rstd, dx_out.contiguous(), dy.contiguous(), dh, dx, dgate,
                              dw_post, dw_pre, low, stream=torch.cuda.current_stream(h.device))
        return dh, dx, dgate, dw_post.to(w_post.dtype), dw_pre.to(w_pre.dtype), None


def _normed(norm, h, x, gate, w_post, w_pre):
    """(x_out, y); what a backward reads is made only where gradients are on."""
    if torch.is_grad_enabled():
        return _Norm.apply(h, x, gate, w_post, w_pre, norm)
    x_out, y = torch.empty_like(x), torch.empty_like(x)
    norm.forward_dev(h, x, gate, w_post, w_pre, x_out, y, stream=torch.cuda.current_stream(x.device))
    return x_out, y


class FrameBlocks:
    """`layers` blocks of `channels` channels over frames of rows x columns tokens; a token sees
    its own frame, the `back` frames before it and the first `sinks` ones.

    Handles keep workspaces, so what may run at the same time has handles of its own: clip() and
    its backward on each CUDA stream, and each FrameStream. A stream's graphs of clip() share its
    handles, and are not replayed at the same time."""

    def __init__(self, ctx: HipDeformConv, channels: int, q_heads: int, kv_heads: int, head_dim: int, layers: int,
                 rows: int, columns: int, back: int, sinks: int = 1, dtype=torch.bfloat16, seed: int = 0, device="cuda"):
        self.rows, self.columns, self.back, self.sinks = rows, columns, back, sinks
        self.frame_tokens, self.dtype, self.device = rows * columns, dtype, device
        self.split = (q_heads, kv_heads, kv_heads)
        pairs = head_dim // 2
        self.rotary = Rotary(ctx, head_dim, (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3))
        self.freq = self.rotary.frequencies(device=device)
        self.append = CacheAppend(ctx)
        self.new_handles = lambda: (
            FrameAttention(ctx, q_heads, kv_heads, head_dim, self.frame_tokens, back, 0, sinks),
            GatedNorm(ctx, channels, self.frame_tokens, residual_scale=1.0 / math.sqrt(layers)))
        self._handles = {}  # by CUDA stream
        self.channels, self.head_dim = channels, head_dim
        g = torch.Generator().manual_seed(seed)

        def weight(rows, columns):
            return (torch.randn(rows, columns, generator=g) / math.sqrt(rows)).to(dtype).to(device)

        def ones():
            return torch.ones(channels, dtype=dtype, device=device)
        self.first = ones()  # the weights of the first block's norm
        self.layers = [{"qkv": weight(channels, sum(self.split) * head_dim), "back": weight(q_heads * head_dim, channels),
                        "gate": weight(channels, channels), "w_post": ones(), "w_pre": ones()} for _ in range(layers)]

    def _of_this_stream(self):
        key = torch.cuda.current_stream(self.first.device).cuda_stream
        if key not in self._handles:
            self._handles[key] = self.new_handles()
        return self._handles[key]

    @property
    def attention(self) -> FrameAttention:
        return self._of_this_stream()[0]

    @property
    def norm(self) -> GatedNorm:
        return self._of_this_stream()[1]

    def parameters(self):
        return [self.first] + [w for layer in self.layers for w in layer.values()]

    def heads(self, qkv):
        """The queries, keys and values of a packed projection, as they lie."""
        return qkv.view(len(qkv), sum(self.split), self.head_dim).split(self.split, 1)

    def _start(self, x, norm):
        """The first block's input: the norm of x, a closed gate before it."""
        closed = torch.zeros(len(x) // self.frame_tokens, self.channels, dtype=x.dtype, device=x.device)
        return _normed(norm, x, x, closed, self.first, self.first)

    def clip(self, x, style, clips: int = 1):
        """x: [clips * frames * rows * columns][channels]; style: [clips * frames][channels], which
        the gates come from. The output of the last block's norm, differentiable."""
        longest = len(x) // clips
        positions = frame_positions(0, longest // self.frame_tokens, self.rows, self.columns, x.device).repeat(clips, 1)
        norm = self.norm
        x, y = self._start(x, norm)
        for w in self.layers:
            h = _Attend.apply(y @ w["qkv"], self, positions, longest) @ w["back"]
            x, y = _normed(norm, h, x, style @ w["gate"], w["w_post"], w["w_pre"])
        return y

    def stream(self, streams: int, frames: int, page_tokens: int = 16) -> "FrameStream":
        """Serving state of this many streams of at most `frames` frames."""
        return FrameStream(self, streams, frames, page_tokens)


class FrameStream:
    """The paged caches of a set of streams that take one frame each at a time."""

    def __init__(self, blocks: FrameBlocks, streams: int, frames: int, page_tokens: int):
        if blocks.back < 0:
            raise ValueError("streams need a window with an end: back of zero or more")
        if blocks.frame_tokens % page_tokens:
            raise ValueError(f"{page_tokens} tokens a page do not divide a frame of {blocks.frame_tokens}")
        self.blocks, self.streams, self.time, self.frames = blocks, streams, 0, frames
        self.attention, self.norm = blocks.new_handles()
        per_frame = blocks.frame_tokens // page_tokens
        kept = min(frames, blocks.sinks + blocks.back + 1)
        # A frame past the sinks lies where the one that has just left its window was.
        slot = [f if f < blocks.sinks else blocks.sinks + (f - blocks.sinks) % (blocks.back + 1) for f in range(frames)]
        pages = (torch.tensor(slot)[:, None] * per_frame + torch.arange(per_frame)).reshape(1, -1)
        self.table = (pages + kept * per_frame * torch.arange(streams)[:, None]).to(torch.int32).to(blocks.device)
        shape = (streams * kept * per_frame, page_tokens, blocks.split[1], blocks.head_dim)
        self.pages = [tuple(torch.empty(shape, dtype=blocks.dtype, device=blocks.device) for _ in range(2))
                      for _ in blocks.layers]
        n = blocks.frame_tokens
        self.cu_q = (torch.arange(streams + 1) * n).to(torch.int32).to(blocks.device)
        self.lens = torch.zeros(streams, dtype=torch.int32, device=blocks.device)
        self.positions = frame_positions(0, 1, blocks.rows, blocks.columns, blocks.device).repeat(streams, 1)

    @torch.no_grad()
    def step(self, x, style):
        """One frame of every stream ([streams * rows * columns][channels], style [streams][channels]):
        what clip() gives for it."""
        b, n = self.blocks, self.blocks.frame_tokens
        if self.time == self.frames:
            raise ValueError(f"the streams have had their {self.frames} frames")
        self.time += 1
        self.lens += n
        stream = torch.cuda.current_stream(x.device)
        x, y = b._start(x, self.norm)
        for w, (k_pages, v_pages) in zip(b.layers, self.pages):
            q, k, v = b.heads(y @ w["qkv"])
            turned = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            out = torch.empty_like(turned)
            b.append.run_dev(k, v, k_pages, v_pages, self.table, self.cu_q, self.lens, b.rotary, self.positions, b.freq,
                             q, turned, stream=stream)
            self.attention.paged_dev(turned, k_pages, v_pages, self.table, self.cu_q, self.lens, out, max_q=n,
                                     max_kv=self.time * n, stream=stream)
            x, y = _normed(self.norm, out.flatten(1) @ w["back"], x, style @ w["gate"], w["w_post"], w["w_pre"])
        self.positions[:, 0] += 1
        return y


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dtype", choices=("f16", "bf16", "f32"), default="bf16")
    ap.add_argument("--frames", type=int, default=12)
    ap.add_argument("--rows", type=int, default=16)
    ap.add_argument("--columns", type=int, default=16)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--back", type=int, default=3)
    ap.add_argument("--steps", type=int, default=5)
    args = ap.parse_args(argv)
    dtype = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[args.dtype]
    blocks = FrameBlocks(HipDeformConv(0), 512, 8, 4, 64, args.layers, args.rows, args.columns, args.back, dtype=dtype)
    g = torch.Generator().manual_seed(1)

    def data(rows):
        return torch.randn(rows, 512, generator=g).to(dtype).cuda()
    x, target = data(args.frames * blocks.frame_tokens), data(args.frames * blocks.frame_tokens)
    style = data(args.frames)
    for p in blocks.parameters():
        p.requires_grad_()
    for step in range(args.steps):
        loss = (blocks.clip(x, style).float() - target.float()).square().mean()
        (512 * loss).backward()  # summed over channels: gradients of a size that FP16 holds
        with torch.no_grad():
            for p in blocks.parameters():
                p -= (0.005 * p.grad.float()).to(p.dtype)
                p.grad = None
        print(f"step {step}: loss {loss.item():.5f}", flush=True)
    with torch.no_grad():
        whole = blocks.clip(x, style).view(args.frames, blocks.frame_tokens, 512)
    serving = blocks.stream(1, args.frames, next(p for p in (64, 16, 4, 1) if blocks.frame_tokens % p == 0))
    frames = x.view(args.frames, blocks.frame_tokens, 512)
    got, times = [], []
    for f, s in zip(frames, style):
        torch.cuda.synchronize()
        start = time.perf_counter()
        got.append(serving.step(f.contiguous(), s[None]))
        torch.cuda.synchronize()
        times.append(time.perf_counter() - start)
    got, each = torch.stack(got), sorted(times)[len(times) // 2]
    off = ((got - whole).double().norm() / whole.double().norm()).item()
    print(f"{args.frames} frames streamed, {each * 1e6:.0f} us a frame (median); against the whole clip: relative difference {off:.1e}")
    # Two orders of the same sums: a few roundings of each block apart.
    return 0 if off < args.layers * {"f16": 2.0**-8, "bf16": 2.0**-5, "f32": 2.0**-18}[args.dtype] else 1


if __name__ == "__main__":
    sys.exit(main())
