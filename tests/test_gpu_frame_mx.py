"""The microscaled cache on the GPU: what an append keeps, what a read gives back, and attention over
its pages, against the definitions in 64 bits."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

TYPES = {"f16": "float16", "bf16": "bfloat16", "f32": "float32"}


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


def tables(torch, lens, page, seed=5, spare=1):
    """A page table for these lengths, in a random order, and how many pages there are."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    pages = sum(used) + 2
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(max(used), 1) + spare), -1, dtype=torch.int32)
    at = 0
    for row, n in zip(table, used):
        row[:n] = order[at:at + n]
        at += n
    return table, pages


# (type, q heads, kv heads, dim, page, new tokens, lengths with them, pairs (None: no rotation), interleaved)
APPEND = [
    ("bf16", 4, 2, 64, 16, [1, 1, 1], [1, 17, 16], (16, 8, 8), False),
    ("f16", 2, 2, 128, 64, [40, 0, 3, 70], [100, 5, 3, 70], (24, 20, 20), False),
    ("f32", 3, 1, 32, 4, [9, 2], [9, 30], (4, 3, 3), False),  # pairs that are no whole chunks, channels that pass
    ("bf16", 0, 2, 64, 16, [5], [21], None, False),
    ("f16", 2, 1, 96, 8, [11, 33], [11, 40], (16, 16, 16), True),
    ("bf16", 5, 3, 160, 1, [7], [9], (1, 2, 2), True),
    ("f32", 2, 2, 256, 32, [130], [200], (64, 32, 32), False),
    ("bf16", 8, 8, 64, 64, [300, 1], [777, 1], (32, 0, 0), False),
    ("f16", 1, 1, 32, 8, [0, 1, 3] * 45, [0, 9, 3] * 45, (8, 4, 4), False),  # more sequences than a wave has lanes
]


def _append_inputs(torch, case, fa, ctx, odd):
    name, hq, hk, dim, page, new, lens, pairs, interleaved = case
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(3)
    gap = 2  # rows of no sequence in front, one behind
    cu = [gap]
    for n in new:
        cu.append(cu[-1] + n)
    tokens = cu[-1] + 1
    width = (hq + 2 * hk) * dim
    whole = (torch.randn(tokens, width + odd, generator=g) * torch.exp2(torch.randint(-4, 5, (tokens, 1), generator=g))).to(dtype)
    heads = whole[:, odd:].unflatten(1, (hq + 2 * hk, dim)).cuda() if not odd else whole.cuda()[:, odd:].unflatten(1, (hq + 2 * hk, dim))
    q, k, v = heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:]
    pos = torch.randint(-50, 400, (tokens, 3), generator=g, dtype=torch.int32)
    table, pages = tables(torch, lens, page)
    rotary = None if pairs is None else fa.Rotary(ctx, dim, pairs, interleaved)
    return dtype, q if hq else None, k, v, cu, pos, table, pages, rotary


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}-{c[1]}.{c[2]}x{c[3]}-p{c[4]}-{c[5][:4]}")
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("odd", [0, 1])
def test_append(fa, gpu_ctx, case, bits, odd):
    import torch

    import frame_attention_reference as ref
    import frame_mx_reference as mx

    name, hq, hk, dim, page, new, lens, pairs, interleaved = case
    print("case: append", case, bits, odd, flush=True)
    dtype, q, k, v, cu, pos, table, pages, rotary = _append_inputs(torch, case, fa, gpu_ctx, odd)
    cache = fa.MxPages.zeros(pages, page, hk, dim, bits)
    for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        t.fill_(0x5A)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    freq = rotary and rotary.frequencies(100.0)
    q_out = None if q is None else torch.zeros_like(q)
    turn = {} if rotary is None else dict(rotary=rotary, positions=pos.cuda(), freq=freq)
    fa.CacheAppend(gpu_ctx).run_mx_dev(k, v, cache, table.cuda(), i32(cu), i32(lens), q=q, q_out=q_out, **turn)
    torch.cuda.synchronize()
    if q is not None:
        want = torch.zeros_like(q)
        if rotary is None:
            want[cu[0]:cu[-1]] = q[cu[0]:cu[-1]]
        else:
            rotary.run_dev(q, pos.cuda(), freq, want)
            want[:cu[0]] = 0
            want[cu[-1]:] = 0
        assert torch.equal(q_out, want)
    k, v = k.cpu(), v.cpu()
    turned = k.double() if rotary is None else ref.rotate(k, pos, freq.cpu(), pairs, interleaved, False)
    # |a| + |b| times FP32 cosines and sines (3 ulp each), two products and a sum
    slack = torch.zeros_like(turned)
    if rotary is not None:
        n = sum(pairs)
        first = torch.arange(n) * 2 if interleaved else torch.arange(n)
        second = first + (1 if interleaved else n)
        both = 8 * 2.0**-24 * (k.double().abs()[..., first] + k.double().abs()[..., second])
        slack[..., first], slack[..., second] = both, both
    left = [t.clone() for t in (cache.k.cpu(), cache.k_scales.cpu(), cache.v.cpu(), cache.v_scales.cpu())]
    near, small = mx.HALF[bits]
    for s, n in enumerate(lens):
        rows = slice(cu[s], cu[s + 1])
        at = torch.arange(n - new[s], n)
        which = table[s][at // page].long()
        codes, scales = mx.quantise(v[rows], bits, dtype)
        assert torch.equal(left[2][which, :, at % page], mx.pack(codes, bits).to(torch.uint8))
        assert torch.equal(left[3][which, :, at % page].long(), scales)
        got, e = left[0][which, :, at % page], left[1][which, :, at % page]
        if rotary is None:
            codes, scales = mx.quantise(k[rows], bits, dtype)
            assert torch.equal(got, mx.pack(codes, bits).to(torch.uint8)) and torch.equal(e.long(), scales)
        else:
            x, off = turned[rows], slack[rows]
            top = x.abs().unflatten(-1, (-1, 32)).amax(-1) if n else x[..., :0]
            most = off.unflatten(-1, (-1, 32)).amax(-1) if n else x[..., :0]
            power = torch.pow(2.0, e.double() - 127)
            assert (top - most <= mx.LARGEST[bits] * power).all() and (top + most > mx.LARGEST[bits] * power / 2).all()
            back = mx.values(got, e, bits)
            step = power.repeat_interleave(32, -1)
            assert ((back - x).abs() <= torch.maximum(near * (x.abs() + off), small * step) + off).all()
        for t in left:
            t[which, :, at % page] = 0x5A
    assert all((t == 0x5A).all() for t in left), "more was written than the new tokens"


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("name", list(TYPES))
def test_append_of_any_value(fa, gpu_ctx, name, bits):
    """Zeros, the smallest and the largest numbers, ties, infinities and NaN."""
    import torch

    import frame_mx_reference as mx

    print("case: values", name, bits, flush=True)
    dtype = getattr(torch, TYPES[name])
    info = torch.finfo(dtype)
    g = torch.Generator().manual_seed(1)
    codes = mx.code_values(bits)[: 1 << (bits - 1)]
    codes = codes[torch.isfinite(codes)]
    middle = (codes[1:] + codes[:-1]) / 2
    rows = [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), info.max), torch.full((32,), -info.max),
            torch.full((32,), info.tiny), torch.arange(32) * info.smallest_normal / 64,
            torch.arange(1, 33) * torch.tensor(info.smallest_normal * info.eps)]
    for special in (float("inf"), float("-inf"), float("nan")):
        one = torch.randn(32, generator=g)
        one[7] = special
        rows.append(one)
    near_most = torch.randn(32, generator=g)
    near_most[3], near_most[5] = info.max, info.max * 0.9
    rows.append(near_most)
    for scale in (1.0, 2.0**-6, 2.0**5):
        for part in middle.split(31):
            row = torch.zeros(32, dtype=torch.float64)
            row[0], row[1:1 + len(part)] = codes[-1] * scale, part * scale
            rows.append(row * (1 - 2 * (torch.arange(32) % 2)))
    for e in range(-30, 16):  # a block's largest at and next to where its power of two changes
        for x in (mx.LARGEST[bits] * 2.0**e, mx.LARGEST[bits] * 2.0**e * (1 + info.eps), mx.LARGEST[bits] * 2.0**e * (1 - info.eps)):
            row = torch.randn(32, generator=g).double() * 2.0**e
            row[9] = x
            rows.append(row)
    x = torch.stack([r.double() for r in rows]).to(dtype)
    if len(x) % 2:
        x = torch.cat([x, x[-1:]])
    x = x.view(-1, 1, 64)
    n = len(x)
    cache = fa.MxPages.zeros(n, 1, 1, 64, bits)
    table = torch.arange(n, dtype=torch.int32, device="cuda")[None]
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    fa.CacheAppend(gpu_ctx).run_mx_dev(x.cuda(), x.flip(0).contiguous().cuda(), cache, table, i32([0, n]), i32([n]))
    out = [torch.empty(n, 1, 64, dtype=dtype, device="cuda") for _ in range(2)]
    fa.CacheRead(gpu_ctx).run_dev(cache, table, i32([0, n]), i32([n]), *out)
    torch.cuda.synchronize()
    codes, scales = mx.quantise(x, bits, dtype)
    for want, got, e, back in ((0, cache.k, cache.k_scales, out[0]), (1, cache.v, cache.v_scales, out[1])):
        c, s = (codes.flip(0), scales.flip(0)) if want else (codes, scales)
        assert torch.equal(e.cpu()[:, 0].long(), s)
        assert torch.equal(got.cpu()[:, 0], mx.pack(c, bits))
        exact = mx.values(mx.pack(c, bits), s, bits)
        assert torch.equal(torch.isnan(exact), torch.isnan(back.cpu()))
        assert torch.equal(exact.to(dtype).nan_to_num(1.0, 9.0, -9.0), back.cpu().nan_to_num(1.0, 9.0, -9.0))
        assert not torch.isinf(back).any()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("odd", [0, 1])
def test_read(fa, gpu_ctx, name, bits, odd):
    """Every code under every scale, rounded once; rows that no sequence has stay."""
    import torch

    import frame_mx_reference as mx

    print("case: read", name, bits, odd, flush=True)
    dtype, page, heads, dim = getattr(torch, TYPES[name]), 16, 2, 256
    pages = 8
    cache = fa.MxPages.zeros(pages, page, heads, dim, bits)
    every = torch.arange(256, dtype=torch.uint8)
    cache.k.copy_(every.repeat(bits, 1).flatten()[: dim * bits // 8].expand(cache.k.shape))
    cache.v.copy_(every.flip(0).repeat(bits, 1).flatten()[: dim * bits // 8].expand(cache.v.shape))
    scales = torch.arange(pages * heads * page, dtype=torch.int64).view(pages, heads, page, 1).expand(cache.k_scales.shape) % 256
    cache.k_scales.copy_(scales)
    cache.v_scales.copy_(255 - scales)
    lens, cu = [40, 0, 64], [1, 31, 31, 95]
    table = torch.tensor([[3, 1, 0, -1], [-1, -1, -1, -1], [2, 7, 9, 5]], dtype=torch.int32)  # page 9 is not there
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    out = []
    for _ in range(2):
        whole = torch.full((97, heads * dim + 3 * odd), 7.0, dtype=dtype, device="cuda")
        out.append(whole[:, odd:odd + heads * dim].unflatten(1, (heads, dim)))
    fa.CacheRead(gpu_ctx).run_dev(cache, table.cuda(), i32(cu), i32(lens), *out)
    torch.cuda.synchronize()
    for got, codes, e in ((out[0].cpu(), cache.k.cpu(), cache.k_scales.cpu()), (out[1].cpu(), cache.v.cpu(), cache.v_scales.cpu())):
        want = torch.full((97, heads, dim), 7.0, dtype=dtype)
        for s, (n, a, b) in enumerate(zip(lens, cu, cu[1:])):
            for row in range(a, b):
                at = n - (b - row)
                which = int(table[s, at // page])
                if 0 <= which < pages:
                    want[row] = mx.values(codes[which, :, at % page], e[which, :, at % page], bits).to(dtype)
        assert torch.equal(torch.isnan(want), torch.isnan(got))
        assert torch.equal(want.nan_to_num(1.0, 9.0, -9.0), got.nan_to_num(1.0, 9.0, -9.0))


# (type, head size, q heads, kv heads, page, query lengths, key lengths, frame, back, ahead, sinks)
ATTEND = [
    ("bf16", 64, 2, 2, 16, [1], [64], 1, -1, 0, 0),
    ("f16", 64, 2, 1, 16, [1, 1, 0, 1], [65, 1, 0, 31], 1, -1, 0, 0),  # odd, one, none
    ("bf16", 128, 8, 2, 64, [1, 1, 1], [200, 64, 333], 1, -1, 0, 0),
    ("f16", 128, 3, 1, 8, [70], [170], 7, 2, 0, 1),  # frames that end inside tiles, pages of eight; a group of three
    ("bf16", 64, 8, 1, 32, [5, 3], [200, 131], 1, 40, 0, 3),
    ("f16", 64, 1, 1, 16, [90], [40], 1, -1, 0, 0),  # more queries than keys: the first see nothing
    ("bf16", 64, 2, 2, 16, [4], [0], 1, -1, 0, 0),  # no key at all
    ("f16", 64, 2, 2, 16, [0, 10], [33, 10], 1, -1, -1, 0),  # every key visible
    ("bf16", 128, 2, 2, 16, [150], [150], 10, 1, 1, 0),
    ("bf16", 64, 4, 4, 128, [300], [300], 1, 0, 0, 1),  # itself and the first token
    ("f16", 128, 2, 2, 64, [260], [515], 64, 1, 0, 1),
    ("bf16", 64, 2, 1, 16, [130], [517], 50, 3, 0, 2),
    ("f16", 64, 8, 8, 16, [1], [1200], 1, -1, 0, 0),
    ("bf16", 128, 16, 2, 16, [1, 1], [1500, 700], 1, 1000, 0, 4),
    ("f32", 64, 2, 1, 16, [40, 7], [40, 19], 3, 4, 0, 1),
    ("f32", 32, 2, 2, 4, [33], [33], 1, -1, 0, 0),
    ("bf16", 96, 2, 2, 1, [20], [70], 1, 20, 0, 1),
    ("f16", 256, 2, 1, 2, [20], [50], 1, -1, 0, 0),
    ("bf16", 64, 2, 1, 4, [9], [77], 1, -1, 0, 0),  # pages of fewer than eight
    ("f32", 64, 1, 1, 8, [0, 2, 1] * 50, [3, 2, 20] * 50, 1, -1, 0, 0),  # more sequences than a wave has lanes
    ("bf16", 128, 8, 2, 16, [0, 2, 1] * 50, [3, 2, 20] * 50, 1, -1, 0, 0),
]
IDS = [f"{c[0]}-d{c[1]}-h{c[2]}.{c[3]}-p{c[4]}-q{'.'.join(map(str, c[5][:5]))}-k{'.'.join(map(str, c[6][:5]))}-f{c[7]}w{c[8]}a{c[9]}s{c[10]}"
       for c in ATTEND]


def kept(torch, case, bits, seed=1, std=1.0):
    """Queries, and a cache of random keys and values: (q, cu, table, buffers on the CPU, key and value
    rows of each sequence in 64 bits)."""
    import frame_mx_reference as mx

    name, dim, hq, hk, page, nq, nk, *_ = case
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(seed)
    cu = [2]
    for n in nq:
        cu.append(cu[-1] + n)
    q = (torch.randn(cu[-1] + 1, hq, dim, generator=g) * std).to(dtype)
    table, pages = tables(torch, nk, page)
    buffers, rows = [], []
    for _ in range(2):
        x = [(torch.randn(n, hk, dim, generator=g) * std).to(dtype) for n in nk]
        codes, scales = mx.to_pages(x, table, page, pages, bits, dtype)
        buffers.append((codes, scales))
        rows.append([mx.from_pages(codes, scales, table[s], n, page, bits) for s, n in enumerate(nk)])
    return q, cu, table, [buffers[0][0], buffers[1][0], buffers[0][1], buffers[1][1]], rows


def close(torch, what, got, want, bound):
    if not want.numel():
        return
    got = got.double()
    assert torch.equal(torch.isinf(want), torch.isinf(got)), what
    fine = torch.isfinite(want)
    off = ((got - want).abs()[fine] / (bound[fine] + 1e-30)).max() if fine.any() else 0.0
    assert not torch.isnan(got).any() and float(off) <= 1.0, (what, float(off))


def run_paged(torch, fa, ctx, case, q, cu, table, buffers, lens, **more):
    name, dim, hq, hk, page, nq, nk, frame, back, ahead, sinks = case
    op = fa.FrameAttention(ctx, hq, hk, dim, frame, back, ahead, sinks)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    op.paged_mx_dev(q.cuda(), fa.MxPages(*(b.cuda() for b in buffers)), table.cuda(), i32(cu), i32(lens), out, lse, max_q=max(nq),
                    max_kv=max(nk), **more)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


@pytest.mark.parametrize("case", ATTEND, ids=IDS)
@pytest.mark.parametrize("bits", [8, 4])
def test_attention(fa, gpu_ctx, case, bits):
    import torch

    import frame_attention_reference as ref

    name, dim, hq, hk, page, nq, nk, frame, back, ahead, sinks = case
    print("case: attend", case, bits, flush=True)
    q, cu, table, buffers, rows = kept(torch, case, bits)
    out, lse = run_paged(torch, fa, gpu_ctx, case, q, cu, table, buffers, nk)
    touched = torch.zeros(len(q), dtype=torch.bool)
    for s in range(len(nq)):
        mine = slice(cu[s], cu[s + 1])
        touched[mine] = True
        seen = ref.visible(nq[s], nk[s], frame, back, ahead, sinks)
        for h in range(hq):
            want = ref.attention(q[mine, h], rows[0][s][:, h // (hq // hk)], rows[1][s][:, h // (hq // hk)], seen,
                                 1 / math.sqrt(dim), q.dtype)
            close(torch, f"out of sequence {s}, head {h}", out[mine, h], *want["out"])
            close(torch, f"lse of sequence {s}, head {h}", lse[mine, h], *want["lse"])
    assert torch.isnan(out[~touched]).all() and torch.isnan(lse[~touched]).all(), "rows of no sequence were written"


@pytest.mark.parametrize("case", [ATTEND[i] for i in (3, 4, 10, 11, 13, 14, 16)], ids=lambda c: f"{c[0]}-d{c[1]}-q{c[5]}-k{c[6]}")
@pytest.mark.parametrize("bits", [8, 4])
def test_what_is_not_visible_does_not_matter(fa, gpu_ctx, case, bits):
    """Blocks that read as NaN (and, in FP32 and BF16, codes that read as infinities) where no query of
    a sequence looks, or only some do: rows that do not see them have the same bits."""
    import torch

    import frame_attention_reference as ref

    name, dim, hq, hk, page, nq, nk, frame, back, ahead, sinks = case
    print("case: unseen", case, bits, flush=True)
    q, cu, table, buffers, _ = kept(torch, case, bits)
    want, want_lse = run_paged(torch, fa, gpu_ctx, case, q, cu, table, buffers, nk)
    for s in range(len(nq)):
        if not nq[s]:
            continue
        seen = ref.visible(nq[s], nk[s], frame, back, ahead, sinks)
        some = [j for j in range(nk[s]) if not seen[:, j].all()]
        if not some:
            continue
        j = some[len(some) // 2]
        for which, byte in ((2, 255), (3, 255), (1, 0x7F)):
            if which == 1 and bits == 4:
                continue
            bad = [b.clone() for b in buffers]
            bad[which][int(table[s, j // page]), :, j % page, 0] = byte
            got, got_lse = run_paged(torch, fa, gpu_ctx, case, q, cu, table, bad, nk)
            sees = torch.zeros(len(q), dtype=torch.bool)
            sees[cu[s]:cu[s + 1]] = seen[:, j]
            rows = torch.zeros(len(q), dtype=torch.bool)
            rows[cu[0]:cu[-1]] = True
            assert torch.equal(got[rows & ~sees], want[rows & ~sees]) and torch.equal(got_lse[rows & ~sees], want_lse[rows & ~sees])
            if sees.any():
                hit = got[sees]
                assert torch.isnan(hit).any(-1).all() if which != 2 else torch.isnan(hit).all()


def test_pages_that_are_not_there(fa, gpu_ctx):
    """Keys on missing pages are not visible."""
    import torch

    import frame_attention_reference as ref

    for case in (("bf16", 64, 4, 2, 8, [3], [100], 1, -1, 0, 0), ("f16", 128, 4, 1, 16, [140], [300], 1, 90, 0, 2),
                 ("f32", 64, 4, 2, 8, [3], [100], 1, -1, 0, 0)):
        for bits in (8, 4):
            name, dim, hq, hk, page, nq, nk, frame, back, ahead, sinks = case
            print("case: holes", case, bits, flush=True)
            q, cu, table, buffers, rows = kept(torch, case, bits)
            holes = table.clone()
            gone = torch.zeros(nk[0], dtype=torch.bool)
            for p, value in ((0, -1), (2, 1 << 30), (5, -(1 << 31)), (nk[0] // page, buffers[0].shape[0])):
                holes[0, p] = value
                gone[p * page:(p + 1) * page] = True
            out, lse = run_paged(torch, fa, gpu_ctx, case, q, cu, holes, buffers, nk)
            seen = ref.visible(nq[0], nk[0], frame, back, ahead, sinks) & ~gone
            for h in range(hq):
                want = ref.attention(q[cu[0]:cu[1], h], rows[0][0][:, h // (hq // hk)], rows[1][0][:, h // (hq // hk)], seen,
                                     1 / math.sqrt(dim), q.dtype)
                close(torch, f"head {h}", out[cu[0]:cu[1], h], *want["out"])
                close(torch, f"lse of head {h}", lse[cu[0]:cu[1], h], *want["lse"])
