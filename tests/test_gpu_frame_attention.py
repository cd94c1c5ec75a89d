"""Windowed attention (FrameAttention) against its definition in 64 bits: contiguous and
paged keys, forward and backward, at the lengths, windows, head layouts and strides where it
can go wrong. Bounds come from the roundings on the way (frame_attention_reference)."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


TYPES = {"f16": "float16", "bf16": "bfloat16", "f32": "float32"}

# (type, head size, q heads, kv heads, query lengths, key lengths, frame, back, ahead, sinks)
CASES = [
    ("bf16", 64, 2, 2, [64], [64], 1, -1, 0, 0),  # whole tiles, causal
    ("f16", 64, 2, 1, [65, 1, 0, 31], [65, 1, 0, 31], 1, -1, 0, 0),  # odd, one, none
    ("bf16", 128, 4, 2, [33, 128], [33, 128], 1, 15, 0, 2),  # window and sinks
    ("f16", 128, 3, 1, [70], [70], 7, 2, 0, 1),  # frames that end inside tiles; a group of three
    ("bf16", 64, 8, 1, [5, 3], [200, 131], 1, 40, 0, 3),  # the last queries of long keys
    ("f16", 64, 1, 1, [90], [40], 1, -1, 0, 0),  # more queries than keys: the first see nothing
    ("bf16", 64, 2, 2, [40], [0], 1, -1, 0, 0),  # no key at all
    ("f16", 64, 2, 2, [0, 10], [33, 10], 1, -1, -1, 0),  # no query; every key visible
    ("bf16", 128, 2, 2, [150], [150], 10, 1, 1, 0),  # frames ahead
    ("f16", 64, 2, 2, [129], [129], 16, 0, 0, 0),  # only the own frame
    ("bf16", 64, 4, 4, [300], [300], 1, 0, 0, 1),  # itself and the first token
    ("f16", 128, 2, 2, [260], [260], 64, 1, 0, 1),
    ("bf16", 128, 16, 2, [1, 1, 1], [1, 64, 77], 1, -1, 0, 0),  # single tokens
    ("bf16", 64, 2, 2, [200], [200], 1000, 0, 0, 0),  # one frame longer than all
    ("f16", 64, 2, 1, [130], [517], 50, 3, 0, 2),
    ("bf16", 64, 1, 1, [513], [513], 1, 100, -1, 5),
    ("f32", 64, 2, 1, [40, 7], [40, 19], 3, 4, 0, 1),
    ("f32", 17, 2, 2, [33], [33], 1, -1, 0, 0),
    ("bf16", 40, 2, 2, [70], [70], 1, 20, 0, 1),
    ("f16", 256, 2, 1, [20], [50], 1, -1, 0, 0),
    ("f16", 1, 1, 1, [9], [9], 1, -1, 0, 0),
]
IDS = [f"{c[0]}-d{c[1]}-h{c[2]}.{c[3]}-q{'.'.join(map(str, c[4]))}-k{'.'.join(map(str, c[5]))}-f{c[6]}w{c[7]}a{c[8]}s{c[9]}"
       for c in CASES]


def _starts(lengths, gap):
    """Row ranges with `gap` rows of no sequence in front."""
    cu = [gap]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def _make(torch, case, seed, gap=2, std=1.0, train=True):
    name, dim, hq, hk, nq, nk, *_ = case
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(seed)
    cq, ck = _starts(nq, gap), _starts(nk, gap)
    r = lambda rows, heads: (torch.randn(rows, heads, dim, generator=g) * std).to(dtype)  # noqa: E731
    tq, tk = cq[-1] + 1, ck[-1] + 1  # a spare row at the end too
    d = {"q": r(tq, hq), "k": r(tk, hk), "v": r(tk, hk), "cu_q": torch.tensor(cq, dtype=torch.int32),
         "cu_kv": torch.tensor(ck, dtype=torch.int32)}
    if train:
        d["dout"] = r(tq, hq)
    return d


def _run(torch, fa, ctx, case, d, train, alter=None, **more):
    name, dim, hq, hk, nq, nk, frame, back, ahead, sinks = case
    op = fa.FrameAttention(ctx, hq, hk, dim, frame, back, ahead, sinks)
    g = {n: t.cuda() for n, t in d.items()}
    if alter:
        alter(g)
    nan = float("nan")
    full = lambda like: torch.full(like.shape, nan, dtype=like.dtype, device="cuda")  # noqa: E731
    got = {"out": full(g["q"]), "lse": torch.full(g["q"].shape[:2], nan, device="cuda")}
    kw = dict(cu_q=g["cu_q"], cu_kv=g["cu_kv"], max_q=max(nq), max_kv=max(nk), **more)
    op.forward_dev(g["q"], g["k"], g["v"], got["out"], got["lse"], **kw)
    if train:
        got.update(dq=full(g["q"]), dk=full(g["k"]), dv=full(g["v"]))
        op.backward_dev(g["q"], g["k"], g["v"], got["out"], got["lse"], g["dout"], got["dq"], got["dk"], got["dv"], **kw)
    torch.cuda.synchronize()
    return {n: t.cpu() for n, t in got.items()}


def _compare(torch, got, case, d, train):
    import frame_attention_reference as ref

    name, dim, hq, hk, nq, nk, frame, back, ahead, sinks = case
    dtype, group, scale = getattr(torch, TYPES[name]), hq // hk, 1 / math.sqrt(dim)
    cq, ck = d["cu_q"].tolist(), d["cu_kv"].tolist()
    touched_q, touched_k = torch.zeros(len(d["q"]), dtype=torch.bool), torch.zeros(len(d["k"]), dtype=torch.bool)
    for s in range(len(nq)):
        rq, rk = slice(cq[s], cq[s + 1]), slice(ck[s], ck[s + 1])
        touched_q[rq], touched_k[rk] = True, True
        seen = ref.visible(nq[s], nk[s], frame, back, ahead, sinks)
        for kh in range(hk):
            sums = {n: (0.0, 0.0) for n in ("dk", "dv")}
            for h in range(kh * group, (kh + 1) * group):
                want = ref.attention(d["q"][rq, h], d["k"][rk, kh], d["v"][rk, kh], seen, scale, dtype,
                                     d["dout"][rq, h] if train else None)
                for n in ("out", "lse") + (("dq",) if train else ()):
                    _close(torch, f"{n} of sequence {s}, head {h}", got[n][rq, h], *want[n])
                if train:
                    sums = {n: (a + want[n][0], b + want[n][1]) for n, (a, b) in sums.items()}
            if train:
                for n, (value, bound) in sums.items():
                    _close(torch, f"{n} of sequence {s}, key head {kh}", got[n][rk, kh], value, bound)
    for n in got:  # rows of no sequence are as they were
        rows = ~(touched_k if n in ("dk", "dv") else touched_q)
        assert torch.isnan(got[n][rows]).all(), f"{n}: rows of no sequence were written"


def _close(torch, what, got, want, bound):
    if not want.numel():
        return
    got = got.double()
    infinite = torch.isinf(want)
    assert torch.equal(got[infinite], want[infinite]), what
    off = ((got - want).abs() / (bound + 1e-7 * bound.max()))[~infinite]
    assert not len(off) or float(off.max()) <= 1.0, f"{what}: {float(off.max()):.3f} of the bound"


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_training_step(fa, gpu_ctx, case):
    import torch

    print("case: training step", case, flush=True)
    d = _make(torch, case, 3)
    _compare(torch, _run(torch, fa, gpu_ctx, case, d, True), case, d, True)


@pytest.mark.parametrize("case", CASES[:4], ids=IDS[:4])
def test_same_bits_again(fa, gpu_ctx, case):
    import torch

    print("case: twice", case, flush=True)
    d = _make(torch, case, 4)
    a, b = (_run(torch, fa, gpu_ctx, case, d, True) for _ in range(2))
    for n in a:
        assert torch.equal(a[n].nan_to_num(-7.0), b[n].nan_to_num(-7.0)), n


def test_packed_and_unaligned_strides(fa, gpu_ctx):
    """Slices of a packed projection, one whose rows start off 16 bytes and one with the heads
    outermost, give the same bits as adjacent tensors (or, on the row kernels, stay in bounds)."""
    import torch

    case = ("bf16", 64, 4, 2, [77, 130], [77, 130], 5, 6, 0, 1)
    print("case: strides", case, flush=True)
    d = _make(torch, case, 5)
    want = _run(torch, fa, gpu_ctx, case, d, True)

    def packed(g):
        whole = torch.cat([g["q"], g["k"], g["v"]], 1)
        g["q"], g["k"], g["v"] = whole[:, :4], whole[:, 4:6], whole[:, 6:]

    def heads_first(g):
        for n in ("q", "k", "v", "dout"):
            g[n] = g[n].transpose(0, 1).contiguous().transpose(0, 1)

    def off(g):
        for n in ("q", "k", "v"):
            t = torch.zeros(g[n].shape[0], g[n].shape[1] * 64 + 3, dtype=g[n].dtype, device="cuda")
            u = t[:, 1:1 + g[n].shape[1] * 64].unflatten(1, (-1, 64))
            u.copy_(g[n])
            g[n] = u

    for change in (packed, heads_first):
        got = _run(torch, fa, gpu_ctx, case, d, True, change)
        for n in want:
            assert torch.equal(got[n].nan_to_num(-7.0), want[n].nan_to_num(-7.0)), (change.__name__, n)
    _compare(torch, _run(torch, fa, gpu_ctx, case, d, True, off), case, d, True)


def test_equal_runs_without_index_arrays(fa, gpu_ctx):
    import torch

    case = ("f16", 64, 2, 2, [50, 50, 50], [50, 50, 50], 1, -1, 0, 0)
    print("case: equal runs", flush=True)
    d = _make(torch, case, 6, gap=0)
    d = {n: (t[:150] if n in ("q", "k", "v", "dout") else t) for n, t in d.items()}
    want = _run(torch, fa, gpu_ctx, case, d, False)
    op = fa.FrameAttention(gpu_ctx, 2, 2, 64)
    g = {n: t.cuda() for n, t in d.items()}
    out = torch.empty_like(g["q"])
    op.forward_dev(g["q"], g["k"], g["v"], out, max_q=50, max_kv=50)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want["out"])


@pytest.mark.parametrize("name,dim", [("bf16", 64), ("f16", 128), ("f16", 40), ("f32", 64)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_what_is_not_visible_does_not_matter(fa, gpu_ctx, name, dim, poison):
    """NaN, infinities and the type's lowest value in keys, values, queries and gradients reach
    only the rows that see them: the others have the bits that they have without."""
    import torch

    case = (name, dim, 2, 1, [100], [100], 1, 30, 0, 2)
    print("case: poison", case, poison, flush=True)
    dtype = getattr(torch, TYPES[name])
    value = torch.finfo(dtype).min if poison == "lowest" else poison
    clean = _make(torch, case, 7, gap=0)
    want = _run(torch, fa, gpu_ctx, case, clean, True)
    import frame_attention_reference as ref

    seen = ref.visible(100, 100, 1, 30, 0, 2)
    at = 45  # in the middle of a tile; seen by the queries 45 .. 75
    for which in ("k", "v"):
        d = {n: t.clone() for n, t in clean.items()}
        d[which][at, 0, dim // 3] = value
        got = _run(torch, fa, gpu_ctx, case, d, True)
        away = ~seen[:, at]
        for n in ("out", "lse", "dq"):
            assert torch.equal(got[n][:100][away], want[n][:100][away]), (which, n)
        reached = seen[~away].any(0)  # keys that an affected query sees too
        for n in ("dk", "dv"):
            assert torch.equal(got[n][:100][~reached], want[n][:100][~reached]), (which, n)
        if poison != "lowest":
            assert not torch.isfinite(got["out"][:100][~away].float()).all(1).all(), which
    for which in ("q", "dout"):
        d = {n: t.clone() for n, t in clean.items()}
        d[which][at, 1, dim // 3] = value
        got = _run(torch, fa, gpu_ctx, case, d, True)
        away = ~seen[at]
        rows = torch.arange(100) != at
        for n in ("dk", "dv"):
            assert torch.equal(got[n][:100][away], want[n][:100][away]), (which, n)
        for n in ("out", "lse", "dq"):
            assert torch.equal(got[n][:100][rows], want[n][:100][rows]), (which, n)
        if poison != "lowest" and which == "dout":
            assert not torch.isfinite(got["dv"][:100][~away].float()).all()


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_scores_of_any_size(fa, gpu_ctx, name):
    """Scores up to several hundred and far below, gradients from 2^-12 to 2^8: the softmax's
    running maximum and the FP16 products' scales hold them."""
    import torch

    case = (name, 64, 2, 2, [160], [160], 1, -1, 0, 0)
    print("case: sizes", name, flush=True)
    for seed, std, grad in ((1, 6.0, 1.0), (2, 0.01, 2.0**-12), (3, 1.0, 2.0**8)):
        d = _make(torch, case, seed)
        d["q"], d["k"] = (d["q"] * std).to(d["q"].dtype), (d["k"] * std).to(d["k"].dtype)
        d["dout"] = (d["dout"] * grad).to(d["dout"].dtype)
        _compare(torch, _run(torch, fa, gpu_ctx, case, d, True), case, d, True)


@pytest.mark.parametrize("name,dim", [("bf16", 64), ("f16", 64), ("f32", 8)])
def test_gradients_against_differences(fa, gpu_ctx, name, dim):
    """Central differences of the 64-bit loss sum(out * dout) along random directions."""
    import torch

    import frame_attention_reference as ref

    case = (name, dim, 1, 1, [37], [45], 3, 4, 0, 1)
    print("case: differences", case, flush=True)
    d = _make(torch, case, 8, gap=0)
    got = _run(torch, fa, gpu_ctx, case, d, True)
    seen, scale = ref.visible(37, 45, 3, 4, 0, 1), 1 / math.sqrt(dim)
    dtype = getattr(torch, TYPES[name])
    x = {"q": d["q"][:37, 0].double(), "k": d["k"][:45, 0].double(), "v": d["v"][:45, 0].double()}
    do = d["dout"][:37, 0].double()
    want = ref.attention(x["q"], x["k"], x["v"], seen, scale, dtype, do)
    loss = lambda **kw: (ref.attention(*[kw.get(n, x[n]) for n in "qkv"], seen, scale, dtype)["out"][0] * do).sum()  # noqa: E731
    g = torch.Generator().manual_seed(9)
    for n in "qkv":
        for _ in range(4):
            way = torch.randn(x[n].shape, generator=g, dtype=torch.float64)
            step = 1e-4
            slope = float(loss(**{n: x[n] + step * way}) - loss(**{n: x[n] - step * way})) / (2 * step)
            grad = got["d" + n][:len(way), 0].double()
            bound = float((want["d" + n][1] * way.abs()).sum())
            # the difference quotient's own error: third derivatives times step^2, and 1e-16 / step
            assert abs(float((grad * way).sum()) - slope) <= bound + 1e-5 * (1 + abs(slope)), n


# ---- the paged cache ------------------------------------------------------------------------

def _paged(torch, fa, ctx, case, d, page, spare=3, holes=(), poison=None, lse=True, seed=1):
    """The keys of _make in pages of a shuffled pool, then paged_dev."""
    name, dim, hq, hk, nq, nk, frame, back, ahead, sinks = case
    width = max(1, -(-max(nk) // page))
    used = [-(-n // page) for n in nk]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(used) + spare, generator=g)
    dtype = d["k"].dtype
    kp, vp = (torch.full((sum(used) + spare, page, hk, dim), float("nan") if poison is None else poison, dtype=dtype)
              for _ in range(2))
    table = torch.full((len(nk), width), -1, dtype=torch.int32)
    n, ck = 0, d["cu_kv"].tolist()
    for s, length in enumerate(nk):
        for c in range(used[s]):
            rows = range(c * page, min(length, (c + 1) * page))
            table[s, c] = order[n]
            for i, r in enumerate(rows):
                kp[order[n], i], vp[order[n], i] = d["k"][ck[s] + r], d["v"][ck[s] + r]
            n += 1
    for s, c, entry in holes:
        table[s, c] = entry
    op = fa.FrameAttention(ctx, hq, hk, dim, frame, back, ahead, sinks)
    q = d["q"].cuda()
    got = {"out": torch.full(q.shape, float("nan"), dtype=dtype, device="cuda"),
           "lse": torch.full(q.shape[:2], float("nan"), device="cuda")}
    op.paged_dev(q, kp.cuda(), vp.cuda(), table.cuda(), d["cu_q"].cuda(), torch.tensor(nk, dtype=torch.int32).cuda(),
                 got["out"], got["lse"] if lse else None, max_q=max(nq), max_kv=max(nk))
    torch.cuda.synchronize()
    return {n: t.cpu() for n, t in got.items()}


@pytest.mark.parametrize("page", [1, 16, 128])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_paged(fa, gpu_ctx, case, page):
    """Pages that end inside a tile, NaN in the rows past a sequence's end."""
    import torch

    print("case: paged", case, page, flush=True)
    d = _make(torch, case, 10, train=False)
    _compare(torch, _paged(torch, fa, gpu_ctx, case, d, page), case, d, False)


LONG = [
    ("bf16", 128, 8, 2, [1, 1, 1], [3000, 1, 2049], 1, -1, 0, 0),
    ("f16", 64, 4, 4, [1], [4097], 1, 1500, 0, 70),
    ("bf16", 64, 8, 8, [1, 2, 4], [1025, 640, 999], 64, 3, 0, 1),
    ("f16", 128, 4, 1, [9, 1], [2500, 5], 1, -1, 0, 0),
    ("bf16", 128, 6, 2, [40], [1300], 100, 5, 0, 1),
]


@pytest.mark.parametrize("case", LONG, ids=[f"{c[0]}-d{c[1]}-q{c[4]}-k{c[5]}" for c in LONG])
def test_long_caches_for_few_queries(fa, gpu_ctx, case):
    """Few rows over many keys: the work is split over the keys and joined."""
    import torch

    print("case: long", case, flush=True)
    d = _make(torch, case, 11, train=False)
    _compare(torch, _paged(torch, fa, gpu_ctx, case, d, 64), case, d, False)
    _compare(torch, _run(torch, fa, gpu_ctx, case, d, False), case, d, False)


def test_pages_out_of_the_window_may_be_gone(fa, gpu_ctx):
    """A table entry that is no page hides its tokens: given back pages behind the window change
    nothing, and holes inside it are keys that are not there."""
    import torch

    import frame_attention_reference as ref

    case = ("bf16", 64, 2, 1, [1], [700], 1, 99, 0, 16)
    print("case: gone", flush=True)
    d = _make(torch, case, 12, gap=0, train=False)
    want = _paged(torch, fa, gpu_ctx, case, d, 16)
    gone = [(0, c, e) for c, e in zip(range(1, 37), [-1, 1 << 30, -5] * 12)]
    got = _paged(torch, fa, gpu_ctx, case, d, 16, holes=gone)
    assert torch.equal(got["out"][:1], want["out"][:1]) and torch.equal(got["lse"][:1], want["lse"][:1])
    inside = [(0, 39, -1), (0, 40, 1 << 20)]  # tokens 624 .. 655
    got = _paged(torch, fa, gpu_ctx, case, d, 16, holes=inside)
    seen = ref.visible(1, 700, 1, 99, 0, 16)
    seen[:, 624:656] = False
    for h in range(2):
        r = ref.attention(d["q"][:1, h], d["k"][:700, 0], d["v"][:700, 0], seen, 0.125, torch.bfloat16)
        _close(torch, "out", got["out"][:1, h], *r["out"])
        _close(torch, "lse", got["lse"][:1, h], *r["lse"])
    every = [(0, c, -1) for c in range(44)]
    got = _paged(torch, fa, gpu_ctx, case, d, 16, holes=every)
    assert (got["out"][:1] == 0).all() and torch.isinf(got["lse"][:1]).all()


def test_offsets_past_32_bits(fa, gpu_ctx):
    """A pool of more than 2^32 bytes of keys, the sequence's pages at its far end."""
    import torch

    case = ("bf16", 128, 4, 4, [1], [300], 1, -1, 0, 0)
    print("case: far pages", flush=True)
    d = _make(torch, case, 13, gap=0, train=False)
    page, pages = 64, (5 << 30) // (64 * 4 * 128 * 2)
    kp, vp = (torch.zeros(pages, page, 4, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = [pages - 1, 3, pages - 3, pages // 2 + 1, pages - 2]
    for c, p in enumerate(at):
        n = min(64, 300 - c * 64)
        kp[p, :n], vp[p, :n] = d["k"][c * 64:c * 64 + n].cuda(), d["v"][c * 64:c * 64 + n].cuda()
    op = fa.FrameAttention(gpu_ctx, 4, 4, 128)
    out = torch.empty(1, 4, 128, dtype=torch.bfloat16, device="cuda")
    op.paged_dev(d["q"][:1].cuda(), kp, vp, torch.tensor([at], dtype=torch.int32, device="cuda"), None,
                 torch.tensor([300], dtype=torch.int32, device="cuda"), out)
    torch.cuda.synchronize()
    del kp, vp
    torch.cuda.empty_cache()
    want = _paged(torch, fa, gpu_ctx, case, d, 64)
    assert torch.equal(out.cpu(), want["out"][:1])


# ---- streams, graphs, refusals -----------------------------------------------------------------

def test_another_stream_and_a_graph(fa, gpu_ctx):
    import torch

    case = ("bf16", 64, 4, 2, [130], [130], 1, 50, 0, 4)
    print("case: stream and graph", flush=True)
    d = _make(torch, case, 14, gap=0)
    want = _run(torch, fa, gpu_ctx, case, d, True)
    op = fa.FrameAttention(gpu_ctx, 4, 2, 64, 1, 50, 0, 4)
    g = {n: t.cuda() for n, t in d.items()}
    got = {"out": torch.empty_like(g["q"]), "lse": torch.empty(g["q"].shape[:2], device="cuda"), "dq": torch.empty_like(g["q"]),
           "dk": torch.empty_like(g["k"]), "dv": torch.empty_like(g["v"])}

    def step(stream):
        kw = dict(cu_q=g["cu_q"], cu_kv=g["cu_kv"], max_q=130, max_kv=130, stream=stream)
        op.forward_dev(g["q"], g["k"], g["v"], got["out"], got["lse"], **kw)
        op.backward_dev(g["q"], g["k"], g["v"], got["out"], got["lse"], g["dout"], got["dq"], got["dk"], got["dv"], **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(side)
    side.synchronize()
    for n in got:
        assert torch.equal(got[n][:130].cpu(), want[n][:130]), n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream())
    for _ in range(3):
        for t in got.values():
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for n in got:
            assert torch.equal(got[n][:130].cpu(), want[n][:130]), n


def test_refusals(fa, dcn, gpu_ctx):
    import torch

    E = dcn.DeformConvError
    t = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    op = fa.FrameAttention(gpu_ctx, 4, 2, 64)
    q, k, out = t(8, 4, 64), t(8, 2, 64), t(8, 4, 64)

    def refused(status, call, *a, **kw):
        with pytest.raises(E) as e:
            call(*a, **kw)
        assert e.value.status == status, e.value
        return e.value.message

    shape, argument, count = dcn.INVALID_SHAPE, dcn.INVALID_ARGUMENT, 2
    refused(shape, fa.FrameAttention, gpu_ctx, 3, 2, 64)
    refused(shape, op.forward_dev, t(8, 3, 64), k, k, out)
    refused(shape, op.forward_dev, q, k, t(7, 2, 64), out)
    refused(argument, op.forward_dev, q, k, t(8, 2, 64, dtype=torch.float16), out)
    refused(argument, op.forward_dev, t(8, 4, 64, dtype=torch.float64), k, k, out)
    refused(shape, op.forward_dev, t(8, 4, 128)[..., ::2], k, k, out)
    refused(shape, op.forward_dev, q, k, k, t(8, 1, 64).expand(8, 4, 64))
    refused(shape, op.forward_dev, q, k, k, out, lse=t(4, 8, dtype=torch.float32))
    refused(shape, op.forward_dev, q, k, k, out, cu_q=torch.zeros(2, dtype=torch.int64, device="cuda"))
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    refused(shape, op.forward_dev, q, k, k, out, cu_q=cu, cu_kv=cu[:2])
    refused(shape, op.forward_dev, q, k, k, out, max_q=4, max_kv=5)  # two runs of five keys
    for bad in (dict(frame_tokens=0), dict(sinks=-1)):
        refused(shape, fa.FrameAttention(gpu_ctx, 4, 2, 64, **bad).forward_dev, q, k, k, out)
    big = fa.FrameAttention(gpu_ctx, 1, 1, 257)
    refused(shape, big.forward_dev, t(1, 1, 257), t(1, 1, 257), t(1, 1, 257), t(1, 1, 257))
    pages, table = t(4, 16, 2, 64), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    refused(shape, op.paged_dev, q, t(4, 12, 2, 64), t(4, 12, 2, 64), table, None, lens, out)
    refused(shape, op.paged_dev, q, pages, t(3, 16, 2, 64), table, None, lens, out)
    refused(shape, op.paged_dev, q, pages, pages, table, None, lens[:0], out)
    refused(shape, op.paged_dev, q, pages, pages, table.long().int().t().expand(2, 2), None, lens, out)
    refused(shape, op.paged_dev, q, t(4, 16, 1, 64), t(4, 16, 1, 64), table, None, lens, out)
    # the C entry: null pointers and a short workspace
    import ctypes as C

    from jasnamacos_amd import _lib

    lib = gpu_ctx._lib
    s = op._forward_shape(q, k, k, out, None, None, None, None, None)
    for n in ("dout", "dq"):
        getattr(s, n + "_stride")[:] = q.stride()[:2]
    for n in ("dk", "dv"):
        getattr(s, n + "_stride")[:] = k.stride()[:2]
    p = q.data_ptr()
    assert lib.dcn_attention_forward_dev(None, C.byref(s), p, p, p, None, None, p, None, None, 0, None) == argument
    assert lib.dcn_attention_forward_dev(gpu_ctx.ctx, None, p, p, p, None, None, p, None, None, 0, None) == argument
    assert lib.dcn_attention_forward_dev(gpu_ctx.ctx, C.byref(s), None, p, p, None, None, p, None, None, 0, None) == argument
    assert "q is null" in gpu_ctx.last_error
    assert lib.dcn_attention_forward_dev(gpu_ctx.ctx, C.byref(s), p + 1, p, p, None, None, p, None, None, 0, None) == argument
    need = lib.dcn_attention_workspace_bytes(C.byref(s), fa.PASS_BACKWARD)
    assert need > 0
    assert lib.dcn_attention_backward_dev(gpu_ctx.ctx, C.byref(s), p, p, p, p, p, p, None, None, p, p, p, p, need - 1, None) == count
    assert f"expected {need}" in gpu_ctx.last_error
    assert isinstance(s, _lib.DcnAttentionShape)
