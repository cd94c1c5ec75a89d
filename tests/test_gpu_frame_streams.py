"""The microscaled cache and shared prefixes as they are used: streams over them, continuations of a
stream, captured graphs, other streams, large pools, and the calls that the library refuses."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import frame_attention_reference as ref
from test_gpu_frame_blocks import DTYPES, WIDE, apart, data, make, tolerance
from test_gpu_frame_graphs import replayed

pytestmark = pytest.mark.gpu

ONE = (96, 4, 2, 64, 1, 4, 4, 2, 1)  # one block: what its cache keeps goes by the input alone


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [8, 4])
def test_stream_over_a_microscaled_cache(fa, monkeypatch, name, bits):
    """A stream over microscaled pages against one over pages of the type that hold what a microscaled
    cache would: appended to one, read back, and written there. The keys and values of one block
    go by the input alone, so both hold the same codes, and what differs are roundings behind them (FP16
    rounds what it reads back of blocks below 2^-14 only, which its own pages do too)."""
    print("case: stream", name, bits, flush=True)
    blocks, tokens = make(name, ONE)
    g, dtype, streams, frames = torch.Generator().manual_seed(6), DTYPES[name], 3, 8
    x = data(g, dtype, streams, frames, tokens, ONE[0]).cuda()
    style = data(g, dtype, streams, frames, ONE[0]).cuda()
    serving, twin = blocks.stream(streams, frames, 16, bits), blocks.stream(streams, frames, 16)
    keep = fa.MxPages.zeros(twin.pages[0][0].shape[0], 16, 2, 64, bits)
    read = fa.CacheRead(blocks.append.ctx)
    append = fa.CacheAppend.run_dev

    def through(self, k, v, k_pages, v_pages, table, cu_q, lens, rotary, positions, freq, q, q_out, stream=None):
        self.run_mx_dev(k, v, keep, table, cu_q, lens, rotary, positions, freq, q, q_out, stream=stream)
        k_back, v_back = torch.empty(k.shape, dtype=k.dtype, device="cuda"), torch.empty(v.shape, dtype=k.dtype, device="cuda")
        read.run_dev(keep, table, cu_q, lens, k_back, v_back, stream=stream)
        append(self, k_back, v_back, k_pages, v_pages, table, cu_q, lens, stream=stream)
    for f in range(frames):
        frame = x[:, f].reshape(-1, ONE[0]), style[:, f].contiguous()
        got = serving.step(*frame)
        with monkeypatch.context() as m:
            m.setattr(fa.CacheAppend, "run_dev", through)
            want = twin.step(*frame)
        for a, b in zip(serving.pages[0]._buffers, keep._buffers):
            assert torch.equal(a, b)
        assert apart(got, want.double().cpu()) < tolerance(dtype, ONE), f"frame {f}"


@pytest.mark.parametrize("name,sizes,bits", [("f32", WIDE, 0), ("f16", WIDE, 0), ("bf16", WIDE, 0), ("f32", ONE, 8), ("bf16", ONE, 8), ("f16", ONE, 4)])
@pytest.mark.parametrize("begun", [1, 2, 5])
def test_continuations(name, sizes, bits, begun):
    """Three streams that are the same for `begun` frames, and one that is then continued in three ways.
    A product of another batch size may round another way, and a code then be a step off: few are,
    and a step is 2^-3 of a value (4 bits: 2^-1), so 16 bits' tolerance holds for those too."""
    print("case: continuations", name, sizes, bits, begun, flush=True)
    blocks, tokens = make(name, sizes)
    g, dtype, copies, frames = torch.Generator().manual_seed(7), DTYPES[name], 3, 8
    x = data(g, dtype, copies, frames, tokens, sizes[0]).cuda()
    style = data(g, dtype, copies, frames, sizes[0]).cuda()
    x[:, :begun], style[:, :begun] = x[:1, :begun].clone(), style[:1, :begun].clone()
    apiece, one = blocks.stream(copies, frames, 16, bits), blocks.stream(2, frames, 16, bits)
    if not bits:
        for pages in apiece.pages + one.pages:
            for t in pages:
                t.fill_(math.nan)
    for f in range(begun):
        apiece.step(x[:, f].reshape(-1, sizes[0]), style[:, f].contiguous())
        # The second stream of two is the one continued; the first had other frames.
        one.step(torch.cat([-x[0, f], x[0, f]]), torch.cat([-style[:1, f], style[:1, f]]))
    forks = one.fork(copies, of=1)
    limit = 2 * (tolerance(dtype, sizes) if not bits else tolerance(torch.bfloat16, sizes))
    for f in range(begun, frames):
        one.step(torch.cat([x[0, f], -x[0, f]]), torch.cat([style[:1, f], -style[:1, f]]))  # goes on by itself
        want = apiece.step(x[:, f].reshape(-1, sizes[0]), style[:, f].contiguous())
        got = forks.step(x[:, f].reshape(-1, sizes[0]), style[:, f].contiguous())
        assert apart(got, want.double().cpu()) < limit, f"frame {f}"
    with pytest.raises(ValueError, match="had their"):
        forks.step(x[:, 0].reshape(-1, sizes[0]), style[:, 0].contiguous())


def test_refusals_of_continuations():
    blocks, tokens = make("f32", ONE)
    serving = blocks.stream(2, 4, 16)
    with pytest.raises(ValueError, match="no frame yet"):
        serving.fork(2)
    serving.step(torch.randn(2 * tokens, ONE[0], device="cuda"), torch.randn(2, ONE[0], device="cuda"))
    with pytest.raises(ValueError, match="no stream 2"):
        serving.fork(2, of=2)
    with pytest.raises(ValueError, match="continue another one"):
        serving.fork(2).fork(2)


@pytest.mark.parametrize("args", [["--bits", "8"], ["--bits", "4", "--forks", "3"], ["--forks", "2"]])
def test_command(args, capsys):
    from jasnamacos_amd import frame_blocks

    assert frame_blocks.main(["--dtype", "bf16", "--frames", "6", "--rows", "4", "--columns", "4", "--steps", "1", *args]) == 0
    out = capsys.readouterr().out
    assert "6 frames streamed" in out and ("continuations" in out) == ("--forks" in args)


def cache_of(fa, g, dtype, heads, dim, page, lens, bits, prefix=0):
    """(pages, tables, lengths) of a random cache; the first table is the prefix's if there is one."""
    from test_gpu_frame_mx import tables

    table, pages = tables(torch, ([prefix] if prefix else []) + lens, page)
    if bits:
        cache = fa.MxPages.zeros(pages, page, heads, dim, bits)
        for t in (cache.k, cache.v):
            t.copy_(torch.randint(0, 127 if bits == 8 else 256, t.shape, generator=g, dtype=torch.int64))
        for t in (cache.k_scales, cache.v_scales):
            t.copy_(torch.randint(118, 123, t.shape, generator=g, dtype=torch.int64))
    else:
        cache = tuple(torch.randn(pages, page, heads, dim, generator=g).to(dtype).cuda() for _ in range(2))
    return cache, table.cuda(), i32(*lens)


@pytest.mark.parametrize("bits", [0, 8, 4])
def test_graph_of_a_shared_call(fa, gpu_ctx, bits):
    """Captured, outgrown by larger calls of the same handle, replayed."""
    print("case: graph of a shared call", bits, flush=True)
    g = torch.Generator().manual_seed(1)
    op = fa.FrameAttention(gpu_ctx, 8, 2, 128)

    def call(streams, prefix, keys):
        cache, table, lens = cache_of(fa, g, torch.bfloat16, 2, 128, 16, [keys - s % 3 for s in range(streams)], bits, prefix)
        q = torch.randn(streams, 8, 128, generator=g).bfloat16().cuda()
        out, lse, first, length = torch.empty_like(q), torch.empty(streams, 8, device="cuda"), table[0].contiguous(), i32(prefix)
        return [out, lse], lambda stream=None: op.shared_dev(q, cache, first, length, table[1:], None, lens, out, lse, stream=stream)
    results, small = call(40, 12000, 70)
    assert op._lib and not torch.cuda.is_current_stream_capturing()
    calls = iter([call(*sizes)[1] for sizes in ((50, 13000, 90), (64, 16000, 200), (80, 20000, 400))])
    replayed(small, results, lambda: next(calls)())


def test_graph_of_a_step(fa, gpu_ctx):
    """Append, read back and attention over a microscaled cache in one graph; the lengths grow on the
    device between the replays, and every replay is what the calls give."""
    print("case: graph of a step", flush=True)
    g = torch.Generator().manual_seed(2)
    cache, table, lens = cache_of(fa, g, torch.float16, 4, 64, 16, [200, 150], 8)
    rotary, append, read, op = fa.Rotary(gpu_ctx, 64, (16, 8, 8)), fa.CacheAppend(gpu_ctx), fa.CacheRead(gpu_ctx), fa.FrameAttention(gpu_ctx, 8, 4, 64)
    freq, cu, lens = rotary.frequencies(), i32(0, 2, 4), i32(90, 40)
    packed = torch.randn(4, 16, 64, generator=g).half().cuda()
    q, k, v = packed[:, :8], packed[:, 8:12], packed[:, 12:]
    positions = torch.randint(0, 50, (4, 3), generator=g, dtype=torch.int32).cuda()
    turned, out = torch.empty(4, 8, 64, dtype=torch.float16, device="cuda"), torch.empty(4, 8, 64, dtype=torch.float16, device="cuda")
    k_back, v_back = (torch.empty(4, 4, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    results = [turned, out, k_back, v_back, *cache._buffers]

    def step(stream):
        append.run_mx_dev(k, v, cache, table, cu, lens, rotary, positions, freq, q, turned, stream=stream)
        read.run_dev(cache, table, cu, lens, k_back, v_back, stream=stream)
        op.paged_mx_dev(turned, cache, table, cu, lens, out, max_q=2, max_kv=208, stream=stream)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream())
    before = [t.clone() for t in cache._buffers]
    for _ in range(4):
        lens += 7
        packed.mul_(-0.75)
        for t, b in zip(cache._buffers, before):
            t.copy_(b)
        step(None)
        torch.cuda.synchronize()
        want = [t.clone() for t in results]
        for t, b in zip(cache._buffers, before):
            t.copy_(b)
        turned.zero_(), out.zero_(), k_back.zero_(), v_back.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip(results, want):
            assert torch.equal(t, w)


def test_two_handles_on_two_streams(fa, gpu_ctx):
    """Calls that run at the same time, a handle each, give what they give alone."""
    print("case: two streams", flush=True)
    g = torch.Generator().manual_seed(3)
    sets = []
    for n in range(2):
        cache, table, lens = cache_of(fa, g, torch.bfloat16, 8, 64, 64, [4000 + 100 * n, 2000], 8)
        q = torch.randn(2, 16, 64, generator=g).bfloat16().cuda()
        sets.append((fa.FrameAttention(gpu_ctx, 16, 8, 64), q, cache, table, lens, torch.empty_like(q)))
    run = lambda s, stream: s[0].paged_mx_dev(s[1], s[2], s[3], None, s[4], s[5], stream=stream)  # noqa: E731
    want = []
    for s in sets:
        run(s, None)
        torch.cuda.synchronize()
        want.append(s[5].clone())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, stream in zip(sets, streams):
            run(s, stream)
    torch.cuda.synchronize()
    assert all(torch.equal(s[5], w) for s, w in zip(sets, want))


@pytest.mark.parametrize("bits", [8, 4])
def test_pools_past_four_gibibytes(fa, gpu_ctx, bits):
    """The last pages of a pool whose buffers end past 2^32 bytes hold what a small pool's do."""
    print("case: large pool", bits, flush=True)
    heads, dim, page, n = 8, 128, 64, 200
    per_page = heads * page * dim * bits // 8
    pages = (1 << 32) // per_page + 40
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(n, heads, dim, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(1, 16, dim, generator=g).bfloat16().cuda()
    append, read, op = fa.CacheAppend(gpu_ctx), fa.CacheRead(gpu_ctx), fa.FrameAttention(gpu_ctx, 16, 8, dim)
    got = []
    for count, table in ((4, i32(0, 1, 2, 3)), (pages, i32(pages - 3, pages - 1, pages - 4, pages - 2))):
        cache = fa.MxPages(*(torch.empty(count, heads, page, w, dtype=torch.uint8, device="cuda") for w in (dim * bits // 8,) * 2 + (dim // 32,) * 2))
        append.run_mx_dev(k, v, cache, table[None], i32(0, n), i32(n))
        back, out, shared = [torch.empty_like(k), torch.empty_like(v)], torch.empty_like(q), torch.empty_like(q)
        read.run_dev(cache, table[None], i32(0, n), i32(n), *back)
        op.paged_mx_dev(q, cache, table[None], None, i32(n), out)
        op.shared_dev(q, cache, table[:2].contiguous(), i32(128), table[None, 2:].contiguous(), None, i32(n - 128), shared)
        torch.cuda.synchronize()
        got.append([*back, out, shared])
        del cache
    assert all(torch.equal(a, b) for a, b in zip(*got))
    torch.cuda.empty_cache()


def test_nothing_to_do(fa, gpu_ctx):
    """No sequences, no queries, no tokens: nothing is written, and nothing refused."""
    cache, table, lens = cache_of(fa, torch.Generator().manual_seed(5), torch.bfloat16, 2, 64, 16, [5], 8)
    op, empty = fa.FrameAttention(gpu_ctx, 4, 2, 64), torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    kv = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, 1, dtype=torch.int32, device="cuda")
    op.paged_mx_dev(empty, cache, table, i32(0, 0), lens, empty)
    op.paged_mx_dev(empty, cache, none, None, torch.empty(0, dtype=torch.int32, device="cuda"), empty)
    op.shared_dev(empty, cache, table[0].contiguous(), i32(5), table, i32(0, 0), lens, empty)
    fa.CacheAppend(gpu_ctx).run_mx_dev(kv, kv, cache, table, i32(0, 0), lens)
    fa.CacheRead(gpu_ctx).run_dev(cache, table, i32(0, 0), lens, kv, kv)
    # A prefix of no pages, and one of none of its tokens.
    q = torch.randn(1, 4, 64).bfloat16().cuda()
    want, got = torch.empty_like(q), torch.empty_like(q)
    op.paged_mx_dev(q, cache, table, None, lens, want)
    for first, n in ((torch.empty(0, dtype=torch.int32, device="cuda"), 0), (table[0].contiguous(), 0), (table[0].contiguous(), -7)):
        got.zero_()
        op.shared_dev(q, cache, first, i32(n), table, None, lens, got)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals(fa, gpu_ctx):
    """In the library itself: pointers that are missing or not aligned, workspaces too small, in-place turns."""
    from jasnamacos_amd.deform_conv import DeformConvError

    cache, table, lens = cache_of(fa, torch.Generator().manual_seed(6), torch.bfloat16, 2, 64, 16, [5], 8)
    q = torch.randn(1, 4, 64).bfloat16().cuda()
    with pytest.raises(DeformConvError, match="different types, key heads or head sizes"):
        fa.FrameAttention(gpu_ctx, 4, 4, 64).paged_mx_dev(q, cache, table, None, lens, torch.empty_like(q))
    with pytest.raises(DeformConvError, match="out rows overlap"):
        fa.FrameAttention(gpu_ctx, 4, 2, 64).paged_mx_dev(q, cache, table, None, lens, torch.empty(1, 1, 64, dtype=q.dtype, device="cuda").expand(1, 4, 64))
    with pytest.raises(DeformConvError, match="exceeds q_tokens"):
        fa.FrameAttention(gpu_ctx, 4, 2, 64).paged_mx_dev(q, cache, table, None, lens, torch.empty_like(q), max_q=2)
    with pytest.raises(DeformConvError, match="prefix max_tokens"):
        fa.FrameAttention(gpu_ctx, 4, 2, 64).shared_dev(q, cache, table[0].contiguous(), i32(1), table, None, lens, torch.empty_like(q), max_prefix=1000)
    rotary = fa.Rotary(gpu_ctx, 64, (16, 8, 8))
    k = torch.randn(1, 2, 64).bfloat16().cuda()
    with pytest.raises(DeformConvError, match="q_out is q"):
        fa.CacheAppend(gpu_ctx).run_mx_dev(k, k, cache, table, i32(0, 1), lens, rotary, torch.zeros(1, 3, dtype=torch.int32, device="cuda"),
                                           rotary.frequencies(), q, q)
    lib, at = gpu_ctx._lib, lambda t: t.data_ptr()  # noqa: E731
    shape = fa._ATTENTION.pack(1, 1, 4, 2, 64, 1, -1, 0, 0, 1, 5, 1.0, 1, 0, 256, 64, 0, 0, 0, 0, 256, 64, *[0] * 8)

    def attend(q_at, *buffers, lens_at=None, table_at=None, out_at=None):
        pages = fa._PAGES.pack(cache.k.shape[0], 16, table.shape[1], 2, 64, 1, 8, 0, *buffers)
        status = lib.dcn_attention_pages_dev(gpu_ctx.ctx, shape, pages, None, q_at, None, at(lens) if lens_at is None else lens_at,
                                             at(table) if table_at is None else table_at, at(q) if out_at is None else out_at, None, None, 0, None)
        with pytest.raises(DeformConvError) as e:
            gpu_ctx._check(status)
        return e.value.message
    good = [at(b) for b in cache._buffers]
    assert "q is null" in attend(None, *good)
    assert "q is not aligned" in attend(at(q) + 1, *good)
    for n, name in enumerate(("k codes", "v codes", "k_scales", "v_scales")):
        assert f"{name} is null" in attend(at(q), *good[:n], 0, *good[n + 1:])
        assert f"{name} is not aligned" in attend(at(q), *good[:n], good[n] + 1, *good[n + 1:])
    assert "kv_lens is not aligned" in attend(at(q), *good, lens_at=at(lens) + 2)
    assert "table is null" in attend(at(q), *good, table_at=C.c_void_p(0))
    # A workspace that is missing, too small, or not aligned.
    shape = fa._ATTENTION.pack(1, 1, 4, 2, 64, 1, -1, 0, 0, 1, 60000, 1.0, 1, 0, 256, 64, 0, 0, 0, 0, 256, 64, *[0] * 8)
    pages = fa._PAGES.pack(cache.k.shape[0], 16, 4000, 2, 64, 1, 8, 0, *good)
    need = lib.dcn_attention_pages_workspace_bytes(shape, pages, None)
    room = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    for workspace, size, message in ((None, need, "is null"), (at(room), need - 1, f"expected {need}"), (at(room) + 4, need, "not aligned")):
        status = lib.dcn_attention_pages_dev(gpu_ctx.ctx, shape, pages, None, at(q), None, at(lens), at(table), at(q), None, workspace, size, None)
        with pytest.raises(DeformConvError, match=message):
            gpu_ctx._check(status)
    torch.cuda.synchronize()
