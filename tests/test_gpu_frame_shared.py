"""Attention of streams that share a prefix, over 16-bit and 32-bit pages and microscaled ones, against
the definition in 64 bits and against the same keys without a prefix."""
from __future__ import annotations

import math

import pytest

from test_gpu_frame_mx import TYPES, close, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


# (type, head size, q heads, kv heads, page, prefix, query lengths, own lengths, frame, back, ahead, sinks)
CASES = [
    ("bf16", 64, 2, 2, 16, 64, [1, 1], [1, 20], 1, -1, 0, 0),
    ("f16", 64, 2, 1, 16, 77, [1, 1, 0, 1, 1], [5, 1, 0, 31, 0], 1, -1, 0, 0),  # odd lengths, none, a query without own keys
    ("bf16", 128, 8, 2, 64, 500, [1] * 9, [200, 64, 333, 1, 2, 3, 65, 100, 7], 1, -1, 0, 0),
    ("f16", 128, 3, 1, 8, 170, [70, 3], [70, 90], 7, 4, 0, 1),  # frames across the border; pages of eight; a group of three
    ("bf16", 64, 8, 1, 32, 0, [5, 3], [200, 131], 1, 40, 0, 3),  # an empty prefix
    ("f16", 64, 1, 1, 16, 30, [90], [40], 1, -1, 0, 0),  # queries that lie inside the prefix, and before it
    ("bf16", 64, 2, 2, 16, 300, [4, 4], [4, 60], 1, 50, 0, 2),  # some see nothing of the prefix but its sinks
    ("f16", 64, 2, 2, 16, 20, [2, 10], [33, 40], 10, 1, 0, 4),  # sinks that go past the prefix
    ("bf16", 128, 2, 2, 16, 150, [150], [150], 10, 1, 1, 0),
    ("f16", 64, 8, 4, 64, 1024, [64, 64, 64], [64, 128, 192], 64, 7, 0, 1),
    ("bf16", 64, 4, 4, 16, 2000, [1] * 40, list(range(1, 41)), 1, -1, 0, 0),  # many rows
    ("f32", 64, 2, 1, 16, 40, [10, 7], [40, 19], 3, 4, 0, 1),
    ("f32", 32, 2, 2, 4, 33, [3, 1], [33, 1], 1, -1, 0, 0),
    ("bf16", 96, 2, 2, 1, 50, [20], [70], 1, 20, 0, 1),
    ("f16", 256, 2, 1, 2, 50, [2, 2], [5, 6], 1, -1, 0, 0),
    ("bf16", 64, 2, 1, 4, 30, [9], [77], 1, -1, -1, 0),
]
IDS = [f"{c[0]}-d{c[1]}-h{c[2]}.{c[3]}-p{c[4]}-P{c[5]}-q{'.'.join(map(str, c[6][:5]))}-k{'.'.join(map(str, c[7][:5]))}-f{c[8]}w{c[9]}a{c[10]}s{c[11]}"
       for c in CASES]


def make(torch, case, bits, seed=1):
    """(q, cu, prefix table, table, buffers, prefix rows, own rows); bits 0: pages of the type."""
    import frame_mx_reference as mx

    name, dim, hq, hk, page, prefix, nq, nk, *_ = case
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(seed)
    cu = [2]
    for n in nq:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + 1, hq, dim, generator=g).to(dtype)
    whole, pages = tables(torch, [prefix] + nk, page)
    buffers, rows = [[], []], [[], []]
    for part in range(2):
        x = [torch.randn(n, hk, dim, generator=g).to(dtype) for n in [prefix] + nk]
        if bits:
            codes, scales = mx.to_pages(x, whole, page, pages, bits, dtype)
            buffers[0].append(codes)
            buffers[1].append(scales)
            rows[part] = [mx.from_pages(codes, scales, whole[s], len(t), page, bits) for s, t in enumerate(x)]
        else:
            pool = torch.randn(pages, page, hk, dim, generator=g).to(dtype)
            for s, t in enumerate(x):
                at = torch.arange(len(t))
                pool[whole[s][at // page].long(), at % page] = t
            buffers[0].append(pool)
            rows[part] = [t.double() for t in x]
    return q, cu, whole[0].contiguous(), whole[1:].contiguous(), buffers[0] + buffers[1], rows


def run(torch, fa, ctx, case, data, op=None, buffers=None, prefix_table=None, table=None, **more):
    name, dim, hq, hk, page, prefix, nq, nk, frame, back, ahead, sinks = case
    q, cu, own_prefix, own_table, own_buffers, _ = data
    op = op or fa.FrameAttention(ctx, hq, hk, dim, frame, back, ahead, sinks)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    on = [b.cuda() for b in (buffers or own_buffers)]
    pages = tuple(on) if len(on) == 2 else fa.MxPages(*on)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    kw = dict(max_q=max(nq), max_kv=max(nk), max_prefix=prefix)
    kw.update(more)
    op.shared_dev(q.cuda(), pages, (own_prefix if prefix_table is None else prefix_table).cuda(), i32([prefix]),
                  (own_table if table is None else table).cuda(), i32(cu), i32(nk), out, lse, **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def visible(torch, prefix, nq, nk, frame, back, ahead, sinks):
    import frame_attention_reference as ref

    return ref.visible(nq, prefix + nk, frame, back, ahead, sinks)


def compare(torch, case, data, out, lse, gone=None):
    import frame_attention_reference as ref

    name, dim, hq, hk, page, prefix, nq, nk, frame, back, ahead, sinks = case
    q, cu, _, _, _, rows = data
    touched = torch.zeros(len(q), dtype=torch.bool)
    for s in range(len(nq)):
        mine = slice(cu[s], cu[s + 1])
        touched[mine] = True
        seen = visible(torch, prefix, nq[s], nk[s], frame, back, ahead, sinks)
        if gone is not None:
            seen = seen & ~gone[s]
        keys, values = (torch.cat([rows[part][0], rows[part][1 + s]]) for part in range(2))
        for h in range(hq):
            want = ref.attention(q[mine, h], keys[:, h // (hq // hk)], values[:, h // (hq // hk)], seen, 1 / math.sqrt(dim), q.dtype)
            close(torch, f"out of sequence {s}, head {h}", out[mine, h], *want["out"])
            close(torch, f"lse of sequence {s}, head {h}", lse[mine, h], *want["lse"])
    assert torch.isnan(out[~touched]).all() and torch.isnan(lse[~touched]).all(), "rows of no sequence were written"


@pytest.mark.parametrize("case", CASES, ids=IDS)
@pytest.mark.parametrize("bits", [0, 8, 4])
def test_shared(fa, gpu_ctx, case, bits):
    import torch

    print("case: shared", case, bits, flush=True)
    data = make(torch, case, bits)
    compare(torch, case, data, *run(torch, fa, gpu_ctx, case, data))


@pytest.mark.parametrize("case", [CASES[i] for i in (2, 3, 9, 11)], ids=lambda c: f"{c[0]}-d{c[1]}-P{c[5]}")
@pytest.mark.parametrize("bits", [0, 8, 4])
def test_loose_bounds(fa, gpu_ctx, case, bits):
    """max_q, max_kv and max_prefix larger than what is there; a prefix length past its bound counts as it."""
    import torch

    print("case: loose", case, bits, flush=True)
    data = make(torch, case, bits)
    wide = torch.cat([data[2], torch.full((9,), -1, dtype=torch.int32)])
    compare(torch, case, data, *run(torch, fa, gpu_ctx, case, data, max_q=4000, max_kv=None, max_prefix=None, prefix_table=wide))
    less = case[:5] + (case[5] - 20,) + case[6:]
    short = data[:5] + ([[r[0][:-20]] + r[1:] for r in data[5]],)
    out, lse = run(torch, fa, gpu_ctx, case, data, max_prefix=case[5] - 20)
    compare(torch, less, short, out, lse)


@pytest.mark.parametrize("case", [CASES[i] for i in (1, 3, 6, 9, 10, 11)], ids=lambda c: f"{c[0]}-d{c[1]}-P{c[5]}")
@pytest.mark.parametrize("bits", [0, 8, 4])
def test_what_is_not_visible_does_not_matter(fa, gpu_ctx, case, bits):
    """NaN in keys and values of the prefix and of one sequence: rows that do not see them have the same bits."""
    import torch

    name, dim, hq, hk, page, prefix, nq, nk, frame, back, ahead, sinks = case
    print("case: unseen", case, bits, flush=True)
    data = make(torch, case, bits)
    q, cu, prefix_table, table, buffers, _ = data
    want, want_lse = run(torch, fa, gpu_ctx, case, data)
    see = [visible(torch, prefix, nq[s], nk[s], frame, back, ahead, sinks) for s in range(len(nq))]
    places = []
    unseen = [j for j in range(prefix) if not all(v[:, j].all() for v in see)]
    if unseen:
        places.append((None, unseen[len(unseen) // 2]))
    for s in range(len(nq)):
        if nk[s] and nq[s]:
            places.append((s, nk[s] // 2))
    for s, j in places[:3]:
        page_of = int((prefix_table if s is None else table[s])[j // page])
        for part in range(2):
            bad = [b.clone() for b in buffers]
            if bits:
                bad[2 + part][page_of, :, j % page, 0] = 255
            else:
                bad[part][page_of, j % page, :, 0] = float("nan")
            got, got_lse = run(torch, fa, gpu_ctx, case, data, buffers=bad)
            sees = torch.zeros(len(q), dtype=torch.bool)
            for t in range(len(nq)):
                if s is None or t == s:
                    sees[cu[t]:cu[t + 1]] = see[t][:, j if s is None else prefix + j]
            rows = torch.zeros(len(q), dtype=torch.bool)
            rows[cu[0]:cu[-1]] = True
            assert torch.equal(got[rows & ~sees], want[rows & ~sees]) and torch.equal(got_lse[rows & ~sees], want_lse[rows & ~sees])
            if sees.any():
                assert torch.isnan(got[sees]).any(-1).all()


@pytest.mark.parametrize("bits", [0, 8, 4])
def test_pages_that_are_not_there(fa, gpu_ctx, bits):
    import torch

    for case in (("bf16", 64, 4, 2, 8, 90, [3, 2], [40, 30], 1, -1, 0, 0), ("f16", 128, 4, 1, 16, 200, [100, 60], [100, 130], 1, 90, 0, 2),
                 ("f32", 64, 4, 2, 8, 90, [3], [40], 1, -1, 0, 0)):
        name, dim, hq, hk, page, prefix, nq, nk, *_ = case
        print("case: holes", case, bits, flush=True)
        data = make(torch, case, bits)
        holes_prefix, holes = data[2].clone(), data[3].clone()
        gone = [torch.zeros(prefix + n, dtype=torch.bool) for n in nk]
        for p, value in ((1, -1), (3, 1 << 30), (prefix // page, -(1 << 31))):
            holes_prefix[p] = value
            for g in gone:
                g[p * page:min((p + 1) * page, prefix)] = True
        holes[0, 2] = data[4][0].shape[0]
        gone[0][prefix + 2 * page:prefix + 3 * page] = True
        compare(torch, case, data, *run(torch, fa, gpu_ctx, case, data, prefix_table=holes_prefix, table=holes), gone=gone)


@pytest.mark.parametrize("bits", [0, 8])
def test_runs_without_starts(fa, gpu_ctx, bits):
    """cu_q None: max_q queries each."""
    import torch

    case = ("bf16", 64, 4, 2, 16, 100, [3, 3, 3], [40, 3, 7], 1, -1, 0, 0)
    print("case: no starts", bits, flush=True)
    data = make(torch, case, bits)
    q = data[0][2:-1].contiguous()
    op = fa.FrameAttention(gpu_ctx, 4, 2, 64)
    on = [b.cuda() for b in data[4]]
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    out, lse = torch.empty_like(q).cuda(), torch.empty(len(q), 4, device="cuda")
    op.shared_dev(q.cuda(), tuple(on) if not bits else fa.MxPages(*on), data[2].cuda(), i32([100]), data[3].cuda(), None, i32(case[7]), out,
                  lse)
    torch.cuda.synchronize()
    pad = torch.full((2,) + out.shape[1:], float("nan"), dtype=out.dtype)
    whole = torch.cat([pad, out.cpu(), pad[:1]])
    lses = torch.cat([torch.full((2, 4), float("nan")), lse.cpu(), torch.full((1, 4), float("nan"))])
    compare(torch, case, data, whole, lses)


# Prefixes long enough, for sequences enough, that they are read once for all of them: the kernels of many rows
# and of single tokens together, those of 32 rows, one after the other, windows that end inside the prefix.
LARGE = [
    ("bf16", 64, 8, 2, 64, 5003, [1] * 64, [1 + 7 * s % 90 for s in range(64)], 1, -1, 0, 0),
    ("f16", 128, 4, 1, 16, 4100, [1] * 70, [1 + 5 * s % 40 for s in range(70)], 1, -1, 0, 0),
    ("bf16", 64, 8, 2, 32, 4000, [1] * 66, [1 + 3 * s % 50 for s in range(66)], 1, 3500, 0, 2),
    ("f16", 128, 8, 8, 8, 2200, [1] * 16, [2 + s for s in range(16)], 1, -1, 0, 0),
    ("bf16", 128, 6, 2, 16, 3000, [s % 12 for s in range(48)], [s % 12 + s for s in range(48)], 1, -1, -1, 0),
    ("f16", 64, 4, 4, 64, 6000, [0 if s % 5 == 3 else 1 for s in range(150)], [s % 3 for s in range(150)], 7, 600, 0, 3),
    ("bf16", 64, 2, 2, 16, 9000, [3] * 40, [s % 7 for s in range(40)], 1, 8000, 0, 0),  # more queries than own keys
]
LARGE_IDS = [f"{c[0]}-d{c[1]}-h{c[2]}.{c[3]}-p{c[4]}-P{c[5]}-n{len(c[6])}-w{c[9]}" for c in LARGE]


def visible_fast(torch, prefix, nq, nk, frame, back, ahead, sinks):
    """As visible, in one go."""
    p = (prefix + nk - nq + torch.arange(nq))[:, None]
    f, fj = torch.div(p, frame, rounding_mode="floor"), (torch.arange(prefix + nk) // frame)[None]
    return (p >= 0) & ((fj <= f + ahead) | (ahead < 0)) & ((fj >= f - back) | (back < 0) | (fj < sinks))


def test_the_masks_agree():
    import torch

    for case in CASES:
        for nq, nk in list(zip(case[6], case[7]))[:3]:
            assert torch.equal(visible_fast(torch, case[5], nq, nk, *case[8:]), visible(torch, case[5], nq, nk, *case[8:]))


@pytest.mark.parametrize("case", LARGE, ids=LARGE_IDS)
@pytest.mark.parametrize("bits", [0, 8, 4])
def test_read_once_for_all(fa, gpu_ctx, monkeypatch, case, bits):
    import torch

    print("case: read once", case, bits, flush=True)
    monkeypatch.setattr("test_gpu_frame_shared.visible", visible_fast)
    name, dim, hq, hk, page, prefix, nq, nk, frame, back, ahead, sinks = case
    if bits == 4 or bits == 8:  # fewer bytes a key: a longer prefix is as many
        case = case[:5] + (prefix * 16 // (4 * bits) + 1,) + case[6:]
    data = make(torch, case, bits)
    op = fa.FrameAttention(gpu_ctx, hq, hk, dim, frame, back, ahead, sinks)
    compare(torch, case, data, *run(torch, fa, gpu_ctx, case, data, op))
    got = [run(torch, fa, gpu_ctx, case, data, op) for _ in range(2)]
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(*got)), "not the same bits again"


@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("case", [LARGE[0], LARGE[4], LARGE[5]], ids=lambda c: f"{c[0]}-d{c[1]}-P{c[5]}")
def test_read_once_and_unseen(fa, gpu_ctx, monkeypatch, case, bits):
    """NaN in the prefix where only some of the rows look, and in a page that is not there for the others."""
    import torch

    name, dim, hq, hk, page, prefix, nq, nk, frame, back, ahead, sinks = case
    print("case: read once, unseen", case, bits, flush=True)
    case = case[:4] + (page, prefix * 16 // (4 * bits) + 1 if bits else prefix) + case[6:]
    prefix = case[5]
    data = make(torch, case, bits)
    q, cu, prefix_table, table, buffers, _ = data
    holes = prefix_table.clone()
    holes[3] = -1
    gone = [torch.zeros(prefix + n, dtype=torch.bool) for n in nk]
    for g in gone:
        g[3 * page:4 * page] = True
    monkeypatch.setattr("test_gpu_frame_shared.visible", visible_fast)
    out, lse = run(torch, fa, gpu_ctx, case, data, prefix_table=holes)
    compare(torch, case, data, out, lse, gone=gone)
    see = [visible_fast(torch, prefix, nq[s], nk[s], frame, back, ahead, sinks) for s in range(len(nq))]
    seen = torch.cat([v[:, :prefix] for v in see]).float().mean(0)
    some = ((seen > 0) & (seen < 1)).nonzero().flatten().tolist()
    for j in ([some[len(some) // 2]] if some else []) + [prefix - 1, 0]:
        bad = [b.clone() for b in buffers]
        at = int(prefix_table[j // page])
        if bits:
            bad[3][at, :, j % page, 0] = 255
        else:
            bad[1][at, j % page, :, 0] = float("nan")
        got, got_lse = run(torch, fa, gpu_ctx, case, data, buffers=bad, prefix_table=holes)
        sees, rows = torch.zeros(len(q), dtype=torch.bool), torch.zeros(len(q), dtype=torch.bool)
        rows[cu[0]:cu[-1]] = True
        for s in range(len(nq)):
            sees[cu[s]:cu[s + 1]] = see[s][:, j]
        assert torch.equal(got[rows & ~sees], out[rows & ~sees]) and torch.equal(got_lse[rows & ~sees], lse[rows & ~sees])
        if sees.any():
            assert torch.isnan(got[sees]).any(-1).all()


def _lies(torch, how, shape, fill):
    """A tensor of this shape [tokens][heads][dim] that lies in memory otherwise, and all of that memory."""
    tokens, heads, dim = shape
    if how == "heads first":
        whole = torch.full((heads, tokens, dim), fill)
        return (lambda w: w.transpose(0, 1)), whole
    if how == "of a wider row":  # as the queries of a packed row of queries, keys and values
        return (lambda w: w[:, :heads]), torch.full((tokens, heads + 5, dim), fill)
    return (lambda w: w[:, :, 1:dim + 1]), torch.full((tokens, heads, dim + 3), fill)  # off 16 bytes: the kernels of any type


@pytest.mark.parametrize("how", ["heads first", "of a wider row", "off 16 bytes"])
@pytest.mark.parametrize("case", [CASES[2], CASES[3], CASES[9]], ids=[IDS[i] for i in (2, 3, 9)])
@pytest.mark.parametrize("bits", [0, 8, 4])
def test_strides(fa, gpu_ctx, case, bits, how):
    import torch

    name, dim, hq, hk, page, prefix, nq, nk, *rest = case
    data = make(torch, case, bits)
    q, cu, prefix_table, table, buffers, _ = data
    view, q_whole = _lies(torch, how, q.shape, 7.0)
    out_view, out_whole = _lies(torch, how, q.shape, 7.0)
    q_whole, out_whole = q_whole.to(q.dtype).cuda(), out_whole.to(q.dtype).cuda()
    view(q_whole).copy_(q)
    out_view(out_whole).fill_(float("nan"))
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    on = [b.cuda() for b in buffers]
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    fa.FrameAttention(gpu_ctx, hq, hk, dim, *rest).shared_dev(
        view(q_whole), tuple(on) if len(on) == 2 else fa.MxPages(*on), prefix_table.cuda(), i32([prefix]), table.cuda(), i32(cu), i32(nk),
        out_view(out_whole), lse, max_q=max(nq), max_kv=max(nk), max_prefix=prefix)
    torch.cuda.synchronize()
    compare(torch, case, data, out_view(out_whole).cpu(), lse.cpu())
    out_view(out_whole).fill_(7.0)
    assert (out_whole == 7.0).all(), "what lies between the rows was written"
