"""Rotary positions with three axes, the append to a paged cache and the gated norms against
their definitions in 64 bits."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


TYPES = {"f16": "float16", "bf16": "bfloat16", "f32": "float32"}


def _positions(torch, g, tokens, far=0):
    p = torch.randint(-50, 400, (tokens, 3), generator=g, dtype=torch.int32)
    return p + torch.tensor([far, 0, -far], dtype=torch.int32)


def _rotary_bound(x, positions, freq, pairs, interleaved, inverse, want, dtype):
    """|a| + |b| times FP32 cosines and sines (3 ulp each), two products and a sum, and one
    rounding to the type."""
    import frame_attention_reference as ref

    ones = ref.rotate(x.abs(), positions * 0, freq, pairs, interleaved, inverse)
    n = sum(pairs)
    size = ones.clone()
    if n:
        import torch

        first = torch.arange(n) * 2 if interleaved else torch.arange(n)
        second = first + (1 if interleaved else n)
        both = ones[..., first] + ones[..., second]
        size[..., first] = both
        size[..., second] = both
    return ref.U[dtype] * want.abs() + 8 * 2.0**-24 * size + ref.TINY[dtype]


ROTARY = [  # (type, tokens, heads, dim, pairs, interleaved, far)
    ("f32", 64, 8, 64, (16, 8, 8), False, 0),
    ("f16", 33, 3, 64, (8, 12, 12), True, 0),
    ("bf16", 1, 1, 128, (64, 0, 0), False, 0),
    ("bf16", 50, 2, 128, (5, 6, 7), False, 0),  # 18 pairs: no whole vectors
    ("f16", 20, 2, 128, (10, 10, 4), True, 0),  # channels that pass
    ("f32", 7, 2, 17, (3, 2, 1), False, 0),
    ("f32", 7, 2, 17, (0, 0, 8), True, 0),
    ("bf16", 9, 2, 64, (0, 0, 0), False, 0),  # nothing turns
    ("f32", 40, 2, 64, (16, 8, 8), False, 2000000000),  # far positions lose nothing
    ("f16", 4097, 5, 64, (12, 10, 10), False, 100000),
]


@pytest.mark.parametrize("case", ROTARY, ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}x{c[3]}-{c[4]}-{c[5]}")
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary(fa, gpu_ctx, case, inverse):
    import torch

    import frame_attention_reference as ref

    name, tokens, heads, dim, pairs, interleaved, far = case
    print("case: rotary", case, inverse, flush=True)
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(1)
    x = torch.randn(tokens, heads, dim, generator=g).to(dtype)
    pos = _positions(torch, g, tokens, far)
    op = fa.Rotary(gpu_ctx, dim, pairs, interleaved)
    freq = op.frequencies(100.0, "cpu")
    want = ref.rotate(x, pos, freq, pairs, interleaved, inverse)
    bound = _rotary_bound(x.double(), pos, freq, pairs, interleaved, inverse, want, dtype)
    got = torch.empty_like(x).cuda()
    op.run_dev(x.cuda(), pos.cuda(), freq.cuda(), got, inverse=inverse)
    torch.cuda.synchronize()
    off = ((got.cpu().double() - want).abs() / (bound + 1e-30)).max()
    assert float(off) <= 1.0, float(off)
    # in place, and over slices of a packed tensor with odd strides
    for spare in (0, 1):
        whole = torch.zeros(tokens, (heads + 1) * dim + spare, dtype=dtype, device="cuda")
        part = whole[:, spare:spare + heads * dim].unflatten(1, (heads, dim))
        part.copy_(x)
        op.run_dev(part, pos.cuda(), freq.cuda(), part, inverse=inverse)
        torch.cuda.synchronize()
        assert torch.equal(part.cpu(), got.cpu())
        assert (whole[:, spare + heads * dim:] == 0).all() and (whole[:, :spare] == 0).all()


def test_rotary_is_undone_by_its_inverse(fa, gpu_ctx):
    """The gradient against differences: the map is linear and orthogonal, so
    <inverse(g), x> = <g, forward(x)>."""
    import torch

    g = torch.Generator().manual_seed(2)
    x, y = (torch.randn(30, 2, 64, generator=g).cuda() for _ in range(2))
    pos = _positions(torch, g, 30).cuda()
    op = fa.Rotary(gpu_ctx, 64, (12, 10, 10))
    freq = op.frequencies()
    a, b = torch.empty_like(x), torch.empty_like(x)
    op.run_dev(x, pos, freq, a)
    op.run_dev(y, pos, freq, b, inverse=True)
    # 3,840 products of about 1 in 64 bits, each factor off by 8 * 2^-24 at most
    assert abs(float((a.double() * y.double()).sum() - (x.double() * b.double()).sum())) <= 16 * 2.0**-24 * 3840 * 4
    op.run_dev(a, pos, freq, b, inverse=True)
    assert float((b - x).abs().max()) <= 32 * 2.0**-24 * float(x.abs().max()) * 2


APPEND = [  # (type, q heads, kv heads, dim, page, new tokens, lengths with them, turned)
    ("bf16", 4, 2, 64, 16, [1, 1, 1], [1, 17, 16], True),
    ("f16", 2, 2, 128, 64, [40, 0, 3, 70], [100, 5, 3, 70], True),
    ("f32", 3, 1, 20, 4, [9, 2], [9, 30], True),
    ("bf16", 0, 2, 64, 16, [5], [21], False),
    ("bf16", 2, 1, 72, 8, [11], [11], True),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}-{c[1]}.{c[2]}x{c[3]}-p{c[4]}-{c[5]}")
@pytest.mark.parametrize("odd", [False, True])
def test_append(fa, gpu_ctx, case, odd):
    import torch

    import frame_attention_reference as ref

    name, hq, hk, dim, page, new, lens, turned = case
    print("case: append", case, odd, flush=True)
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(3)
    gap = 2  # rows of no sequence in front, one behind
    cu = [gap]
    for n in new:
        cu.append(cu[-1] + n)
    tokens = cu[-1] + 1
    width = -(-max(lens) // page) + 1
    pages = sum(-(-n // page) for n in lens) + 2
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    n = 0
    for s, length in enumerate(lens):
        for c in range(-(-length // page)):
            table[s, c] = order[n]
            n += 1
    packed = torch.randn(tokens, (hq + 2 * hk) * dim + odd, generator=g).to(dtype).cuda()
    heads = packed[:, odd:].unflatten(1, (hq + 2 * hk, dim))
    q, k, v = heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:]
    pos = _positions(torch, g, tokens)
    op = fa.Rotary(gpu_ctx, dim, (dim // 8, dim // 8, dim // 8))
    freq = op.frequencies(100.0, "cpu")
    kp, vp = (torch.full((pages, page, hk, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    q_out = torch.full((tokens, hq, dim), 7.0, dtype=dtype, device="cuda") if hq else None
    more = dict(rotary=op, positions=pos.cuda(), freq=freq.cuda()) if turned else {}
    fa.CacheAppend(gpu_ctx).run_dev(k, v, kp, vp, table.cuda(), torch.tensor(cu, dtype=torch.int32).cuda(),
                                    torch.tensor(lens, dtype=torch.int32).cuda(), q=q if hq else None, q_out=q_out, **more)
    torch.cuda.synchronize()

    def want_of(x):
        x = x.cpu()
        if not turned:
            return x.double(), torch.zeros_like(x.double()) + 1e-30
        w = ref.rotate(x, pos, freq, op.pairs, False, False)
        return w, _rotary_bound(x.double(), pos, freq, op.pairs, False, False, w, dtype)

    want_k, want_v = torch.full(kp.shape, 7.0, dtype=torch.float64), torch.full(kp.shape, 7.0, dtype=torch.float64)
    bound = torch.full(kp.shape, 1e-30, dtype=torch.float64)
    ks, kb = want_of(k)
    for s in range(len(new)):
        for i in range(new[s]):
            p = lens[s] - new[s] + i
            at = (int(table[s, p // page]), p % page)
            want_k[at], bound[at], want_v[at] = ks[cu[s] + i], kb[cu[s] + i], v[cu[s] + i].cpu().double()
    assert float(((kp.cpu().double() - want_k).abs() / bound).max()) <= 1.0
    assert torch.equal(vp.cpu().double(), want_v)
    if hq:
        qs, qb = want_of(q)
        inside = slice(gap, cu[-1])
        assert float(((q_out.cpu().double() - qs).abs() / qb)[inside].max()) <= 1.0
        assert (q_out[:gap] == 7).all() and (q_out[cu[-1]:] == 7).all()


def test_append_skips_what_has_no_place(fa, gpu_ctx):
    """Tokens before the sequence's start, past the table and on pages of no pool are not written."""
    import torch

    print("case: append without a place", flush=True)
    one = torch.ones(6, 1, 8, dtype=torch.float16, device="cuda")
    kp, vp = (torch.zeros(3, 4, 1, 8, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[0, -1], [99, 1], [2, 2]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    lens = torch.tensor([5, 1, 20], dtype=torch.int32, device="cuda")  # 3, 4 (no page); -1, 0 (page 99); 18, 19 (past)
    fa.CacheAppend(gpu_ctx).run_dev(one, one, kp, vp, table, cu, lens)
    torch.cuda.synchronize()
    assert float(kp.sum()) == 8 and (kp[0, 3] == 1).all() and float(vp.sum()) == 8
    # index arrays that make no sense write nothing out of place
    cu = torch.tensor([0, 100, -7, 6], dtype=torch.int32, device="cuda")
    fa.CacheAppend(gpu_ctx).run_dev(one, one, kp, vp, table, cu, torch.full((3,), -9, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert float(kp.sum()) == 8


NORM = [  # (type, tokens, channels, gate_tokens, scale, gate, w_post, w_pre, y)
    ("f32", 64, 512, 64, 0.5, True, True, True, True),
    ("bf16", 37, 64, 5, 1.0, True, True, True, True),  # the last gate run is short
    ("f16", 1, 1000, 1, 0.25, True, True, True, True),
    ("bf16", 130, 257, 1, 1.0, True, False, True, True),  # channels of no whole vectors, a gate a token
    ("f16", 50, 1024, 1000, 1.0, True, True, False, True),  # one run longer than all
    ("bf16", 33, 2048, 8, 1.0, False, True, True, True),
    ("f32", 9, 4096, 3, 1.0, True, True, True, True),
    ("bf16", 6, 8192, 2, 1.0, True, True, True, True),
    ("f16", 40, 96, 10, 1.0, False, False, False, False),  # nothing but the first norm
    ("bf16", 700, 8, 100, 1.0, True, True, True, True),
    ("f32", 5, 1, 2, 1.0, True, True, True, True),
]


def _norm_inputs(torch, case, seed):
    name, tokens, c, run, scale, gate, w_post, w_pre, y = case
    dtype = getattr(torch, TYPES[name])
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, mean=0.0, std=1.0: (torch.randn(*s, generator=g) * std + mean).to(dtype)  # noqa: E731
    d = {"h": r(tokens, c, std=2.0), "x": r(tokens, c)}
    d["gate"] = r(-(-tokens // run), c, mean=0.5, std=0.5) if gate else None
    d["w_post"] = r(c, mean=1.0, std=0.2) if w_post else None
    d["w_pre"] = r(c, mean=1.0, std=0.2) if w_pre else None
    d["dx_out"], d["dy"] = r(tokens, c), r(tokens, c) if y else None
    return d


def _norm_run(torch, fa, ctx, case, d, shift=0, keep=True, in_place=False):
    name, tokens, c, run, scale, *_ = case
    op = fa.GatedNorm(ctx, c, run, scale, 1e-5)

    def on(t):
        if t is None:
            return None
        flat = torch.zeros(t.numel() + shift, dtype=t.dtype, device="cuda")[shift:]
        return flat.view(t.shape).copy_(t)

    g = {n: on(t) for n, t in d.items()}
    got = {"x_out": g["x"] if in_place else on(d["x"]), "y": on(d["dy"])}
    rstd = torch.empty(tokens, 2, device="cuda")
    op.forward_dev(g["h"], g["x"], g["gate"], g["w_post"], g["w_pre"], got["x_out"], got["y"], rstd)
    if not keep:
        op = fa.GatedNorm(ctx, c, run, scale, 1e-5)
    got.update(dh=on(d["h"]), dx=on(d["x"]), dgate=on(d["gate"]))
    got.update({"d" + n: torch.empty(c, device="cuda") if d[n] is not None else None for n in ("w_post", "w_pre")})
    op.backward_dev(g["h"], got["x_out"], g["gate"], g["w_post"], g["w_pre"], rstd, g["dx_out"], g["dy"], got["dh"], got["dx"],
                    got["dgate"], got["dw_post"], got["dw_pre"] if d["dy"] is not None else None)
    torch.cuda.synchronize()
    return {n: t.cpu() for n, t in got.items() if t is not None}


def _norm_want(torch, case, d):
    import frame_attention_reference as ref

    name, tokens, c, run, scale, *_ = case
    x = {n: (None if t is None else t.double().requires_grad_(True)) for n, t in d.items() if n not in ("dx_out", "dy")}
    x_out, y = ref.gated_norm(x["h"], x["x"], x["gate"], x["w_post"], x["w_pre"], run, scale, 1e-5)
    outs, grads = ([x_out, y], [d["dx_out"].double(), d["dy"].double()]) if d["dy"] is not None else ([x_out], [d["dx_out"].double()])
    names = [n for n in x if x[n] is not None and (n != "w_pre" or d["dy"] is not None)]
    got = dict(zip(("d" + n for n in names), torch.autograd.grad(outs, [x[n] for n in names], grads)))
    got["x_out"] = x_out.detach()
    if d["dy"] is not None:
        got["y"] = y.detach()
    return got


def _norm_bound(torch, case, d, want, name_of, low):
    """One rounding to the type, and the FP32 steps: rows are sums of c terms (off by c 2^-24 of
    their magnitude at worst, the mean of it 2 sqrt(c) at most taken here as c / 8 + 16), sums
    over tokens as many again. Magnitudes: the largest value that enters an output."""
    import frame_attention_reference as ref

    dtype = getattr(torch, TYPES[case[0]])
    tokens, c, run = case[1], case[2], case[3]
    u = ref.U[dtype]
    step = 2.0**-24 * (c / 8 + 32)
    if not low and dtype != torch.float32:
        step = step + u  # x_out as it was rounded
    value = want[name_of]
    if name_of in ("x_out", "y", "dx"):
        return u * value.abs() + step * value.abs().amax(1, keepdim=True) * 4
    if name_of == "dh":  # a difference: of r1 dn and its mean along n
        t = want["dx"] * case[4]
        for n in ("gate", "w_post"):
            if d[n] is not None:
                w = d[n].double()
                t = t * (w.repeat_interleave(run, 0)[:tokens] if n == "gate" else w)
        t = t / torch.sqrt((d["h"].double() ** 2).mean(1, keepdim=True) + 1e-5)
        return u * value.abs() + step * t.abs().amax(1, keepdim=True) * 4
    # per token terms of the sums: |t| |gate| |n| and the like, at most their largest product
    terms = {"dgate": run, "dw_post": tokens, "dw_pre": tokens}[name_of]
    big = 40.0 * case[4] if name_of != "dw_pre" else 40.0
    return (u if name_of == "dgate" else 0) * value.abs() + (step + 2.0**-24 * terms**0.5 * 4) * big * terms**0.5


@pytest.mark.parametrize("case", NORM, ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}-g{c[3]}")
def test_gated_norm(fa, gpu_ctx, case):
    import torch

    print("case: norm", case, flush=True)
    d = _norm_inputs(torch, case, 4)
    want = _norm_want(torch, case, d)
    got = _norm_run(torch, fa, gpu_ctx, case, d)
    for n, w in want.items():
        bound = _norm_bound(torch, case, d, want, n, True)
        off = ((got[n].double() - w).abs() / (bound + 1e-30)).max()
        assert float(off) <= 1.0, (n, float(off))
    again = _norm_run(torch, fa, gpu_ctx, case, d, in_place=True)
    for n in got:
        assert torch.equal(again[n], got[n]), f"{n} with x_out in x's place"
    odd = _norm_run(torch, fa, gpu_ctx, case, d, shift=1)  # off 16 bytes: element by element
    for n, w in want.items():
        bound = _norm_bound(torch, case, d, want, n, True)
        assert float(((odd[n].double() - w).abs() / (bound + 1e-30)).max()) <= 1.0, n


def test_norm_without_the_low_halves(fa, gpu_ctx):
    """Another handle's backward, or one that ran another forward since, takes x_out as rounded."""
    import torch

    case = NORM[1]
    print("case: norm without low halves", flush=True)
    d = _norm_inputs(torch, case, 5)
    want = _norm_want(torch, case, d)
    got = _norm_run(torch, fa, gpu_ctx, case, d, keep=False)
    for n, w in want.items():
        bound = _norm_bound(torch, case, d, want, n, False)
        assert float(((got[n].double() - w).abs() / (bound + 1e-30)).max()) <= 1.0, n
    # two forwards, then the first one's backward: nothing of the second gets in
    name, tokens, c, run, scale, *_ = case
    op = fa.GatedNorm(gpu_ctx, c, run, scale, 1e-5)
    a = {n: t.cuda() for n, t in d.items()}
    b = {n: t.cuda() for n, t in _norm_inputs(torch, case, 6).items()}
    kept = []
    for t in (a, b):
        x_out, rstd = torch.empty_like(t["x"]), torch.empty(tokens, 2, device="cuda")
        op.forward_dev(t["h"], t["x"], t["gate"], t["w_post"], t["w_pre"], x_out, torch.empty_like(x_out), rstd)
        kept.append((x_out, rstd))
    dh, dx = torch.empty_like(a["x"]), torch.empty_like(a["x"])
    op.backward_dev(a["h"], kept[0][0], a["gate"], a["w_post"], a["w_pre"], kept[0][1], a["dx_out"], a["dy"], dh, dx)
    torch.cuda.synchronize()
    assert torch.equal(dh.cpu(), got["dh"]) and torch.equal(dx.cpu(), got["dx"])


def test_norm_gradients_against_differences(fa, gpu_ctx):
    import torch

    import frame_attention_reference as ref

    case = ("f32", 12, 40, 5, 0.7, True, True, True, True)
    print("case: norm differences", flush=True)
    d = _norm_inputs(torch, case, 7)
    got = _norm_run(torch, fa, gpu_ctx, case, d)
    x = {n: d[n].double() for n in ("h", "x", "gate", "w_post", "w_pre")}

    def loss(**kw):
        x_out, y = ref.gated_norm(*[kw.get(n, x[n]) for n in ("h", "x", "gate", "w_post", "w_pre")], 5, 0.7, 1e-5)
        return float((x_out * d["dx_out"].double()).sum() + (y * d["dy"].double()).sum())

    g = torch.Generator().manual_seed(8)
    for n in x:
        way = torch.randn(x[n].shape, generator=g, dtype=torch.float64)
        slope = (loss(**{n: x[n] + 1e-5 * way}) - loss(**{n: x[n] - 1e-5 * way})) / 2e-5
        # 480 terms of a few units in FP32, and the quotient's third-order error
        assert abs(float((got["d" + n].double() * way).sum()) - slope) <= 1e-4 * (1 + abs(slope)), n


def test_nothing_to_do(fa, gpu_ctx):
    import torch

    e = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    op = fa.Rotary(gpu_ctx, 64, (16, 8, 8))
    op.run_dev(e(0, 4, 64), e(0, 3, dtype=torch.int32), op.frequencies(), e(0, 4, 64))
    n = fa.GatedNorm(gpu_ctx, 64, 4)
    n.forward_dev(e(0, 64), e(0, 64), e(0, 64), e(64), e(64), e(0, 64), e(0, 64), e(0, 2, dtype=torch.float32))
    dw = torch.full((64,), 3.0, device="cuda")
    n.backward_dev(e(0, 64), e(0, 64), e(0, 64), e(64), e(64), e(0, 2, dtype=torch.float32), e(0, 64), e(0, 64), e(0, 64),
                   e(0, 64), e(0, 64), dw, dw.clone())
    torch.cuda.synchronize()
    assert (dw == 0).all()  # the sum over no tokens


def test_refusals(fa, dcn, gpu_ctx):
    import torch

    t = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    i32 = torch.int32

    def refused(status, call, *a, **kw):
        with pytest.raises(dcn.DeformConvError) as e:
            call(*a, **kw)
        assert e.value.status == status, e.value

    shape, argument = dcn.INVALID_SHAPE, dcn.INVALID_ARGUMENT
    op = fa.Rotary(gpu_ctx, 64, (16, 8, 8))
    f, x, p = op.frequencies(), t(4, 2, 64), t(4, 3, dtype=i32)
    refused(shape, fa.Rotary, gpu_ctx, 64, (16, 8))
    refused(shape, fa.Rotary(gpu_ctx, 64, (16, 16, 8)).run_dev, x, p, t(40, dtype=torch.float32), x)
    refused(shape, fa.Rotary(gpu_ctx, 64, (16, -8, 8)).run_dev, x, p, t(16, dtype=torch.float32), x)
    refused(shape, op.run_dev, x, t(4, 2, dtype=i32), f, x)
    refused(argument, op.run_dev, x, p.long(), f, x)
    refused(shape, op.run_dev, x, p, f[:31], x)
    refused(shape, op.run_dev, x, p, f, t(4, 1, 64).expand(4, 2, 64))
    refused(argument, op.run_dev, x, p, f, t(4, 2, 64, dtype=torch.float16))
    refused(argument, op.run_dev, x, p, f, x.double())
    n = fa.GatedNorm(gpu_ctx, 64, 4)
    refused(shape, fa.GatedNorm, gpu_ctx, 64, 0)
    refused(shape, n.forward_dev, t(8, 64), t(7, 64), None, None, None, t(7, 64))
    refused(shape, n.forward_dev, t(8, 64), t(8, 64), t(3, 64), None, None, t(8, 64))
    refused(argument, n.forward_dev, t(8, 64), t(8, 64), None, t(64, dtype=torch.float32), None, t(8, 64))
    refused(shape, n.forward_dev, t(8, 128)[:, ::2], t(8, 64), None, None, None, t(8, 64))
    big = fa.GatedNorm(gpu_ctx, 8193)
    refused(shape, big.forward_dev, t(1, 8193), t(1, 8193), None, None, None, t(1, 8193))
    a = fa.CacheAppend(gpu_ctx)
    kp, table, cu, lens = t(2, 16, 1, 64), t(1, 2, dtype=i32), t(2, dtype=i32), t(1, dtype=i32)
    one = t(1, 1, 64)
    refused(shape, a.run_dev, one, one, t(2, 12, 1, 64), t(2, 12, 1, 64), table, cu, lens)
    refused(shape, a.run_dev, one, one, kp, kp, table, cu[:1], lens)
    refused(shape, a.run_dev, t(1, 2, 64), one, kp, kp, table, cu, lens)
    refused(shape, a.run_dev, one, one, kp, kp, table, cu, lens, rotary=fa.Rotary(gpu_ctx, 32, (4, 4, 4)), positions=t(1, 3, dtype=i32),
            freq=t(12, dtype=torch.float32))
