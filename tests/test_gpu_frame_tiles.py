"""FrameAttention at the sizes that real clips have, where the work is laid out in other ways than for
short calls: 128 rows a workgroup and several workgroups a sequence (forward and query gradients),
their keys in parts, and key gradients whose queries are in parts. Against the definition in 64 bits,
with the bounds of frame_attention_reference."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

TYPES = {"f16": "float16", "bf16": "bfloat16"}

# (type, head size, q heads, kv heads, query lengths, key lengths, frame, back, ahead, sinks)
LENGTHS = [800, 333, 1, 0, 650]  # of 8 heads on 4: 13 x 4 x 5 blocks of 128 rows, more than 256
SHORTER = [400, 257, 0, 31, 390]  # of 8 heads on 2: 13 x 2 x 5, more than 128
CASES = [
    ("bf16", 64, 8, 4, LENGTHS, LENGTHS, 1, 100, 0, 3),  # tiles before the window, and gaps in it
    ("f16", 64, 8, 4, LENGTHS, [900, 333, 70, 5, 650], 64, 2, 1, 1),  # whole frames, one ahead
    ("bf16", 64, 8, 4, LENGTHS, LENGTHS, 1, -1, 0, 0),
    ("f16", 64, 8, 4, LENGTHS, [700, 333, 1, 0, 650], 1, 500, 0, 70),  # queries before the first key
    ("bf16", 128, 8, 2, SHORTER, [700, 257, 5, 31, 390], 50, 3, 0, 2),
    ("f16", 128, 8, 2, SHORTER, SHORTER, 1, -1, 0, 0),
    ("f16", 128, 8, 2, SHORTER, SHORTER, 1, 90, 0, 5),
    ("bf16", 128, 8, 2, SHORTER, SHORTER, 7, 11, -1, 3),  # all that follows
    ("bf16", 64, 2, 2, [300], [5000], 1, -1, 0, 0),  # more than 4,096 keys: in parts
    ("f16", 64, 3, 1, [131, 40], [4500, 4999], 1, 4400, 0, 66),
    ("f16", 128, 3, 1, [129, 16], [3000, 2100], 1, -1, 0, 0),  # more than 2,048
    ("bf16", 128, 2, 2, [200], [2600], 100, 22, 0, 1),
]
# Key gradients in parts: (case, parts of a block of 128 keys, blocks of sinks, their parts).
PARTS = [
    (("bf16", 64, 8, 1, [520], [520], 1, -1, 0, 0), 8, 0, 0),
    (("f16", 64, 8, 1, [520], [520], 1, 200, 0, 4), 5, 1, 8),
    (("bf16", 128, 8, 1, [520, 77], [520, 300], 1, -1, -1, 0), 8, 0, 0),
    (("f16", 128, 8, 1, [520, 333], [520, 400], 1, 200, 0, 140), 5, 2, 8),
    (("bf16", 128, 16, 2, [521], [640], 32, 5, 0, 1), 5, 1, 8),
    (("f16", 128, 4, 2, [1021], [1021], 1, 255, 0, 4), 1, 1, 3),  # the sinks' alone
]


def name_of(case):
    return f"{case[0]}-d{case[1]}-h{case[2]}.{case[3]}-q{case[4][0]}-k{case[5][0]}-f{case[6]}w{case[7]}a{case[8]}s{case[9]}"


def visible(nq, nk, frame, back, ahead, sinks, device="cuda"):
    import torch

    p = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None]
    f, fj = torch.div(p, frame, rounding_mode="floor"), torch.div(j, frame, rounding_mode="floor")
    seen = (p >= 0) & (j >= 0)
    if ahead >= 0:
        seen = seen & (fj <= f + ahead)
    if back >= 0:
        seen = seen & ((fj >= f - back) | (fj < sinks))
    return seen


def starts(lengths):
    import torch

    return torch.tensor([2] + [2 + sum(lengths[:i + 1]) for i in range(len(lengths))], dtype=torch.int32)


def make(case, seed):
    """Tensors on the GPU: two rows of no sequence in front, one behind."""
    import torch

    name, dim, hq, hk, nq, nk = case[:6]
    g = torch.Generator().manual_seed(seed)
    r = lambda rows, heads: torch.randn(rows + 3, heads, dim, generator=g).to(getattr(torch, TYPES[name])).cuda()  # noqa: E731
    return {"q": r(sum(nq), hq), "k": r(sum(nk), hk), "v": r(sum(nk), hk), "dout": r(sum(nq), hq)}


def step(ctx, case, d, paged=None):
    """(outputs, the handle): a training step, or the paged forward at this many tokens a page."""
    import torch

    from jasnamacos_amd.frame_attention import FrameAttention

    name, dim, hq, hk, nq, nk, *window = case
    op = FrameAttention(ctx, hq, hk, dim, *window)
    full = lambda like: torch.full_like(like, math.nan)  # noqa: E731
    got = {"out": full(d["q"]), "lse": torch.full(d["q"].shape[:2], math.nan, device="cuda")}
    cu_q, cu_kv = starts(nq).cuda(), starts(nk).cuda()
    if paged is None:
        kw = dict(cu_q=cu_q, cu_kv=cu_kv, max_q=max(nq), max_kv=max(nk))
        op.forward_dev(d["q"], d["k"], d["v"], got["out"], got["lse"], **kw)
        got.update(dq=full(d["q"]), dk=full(d["k"]), dv=full(d["v"]))
        op.backward_dev(d["q"], d["k"], d["v"], got["out"], got["lse"], d["dout"], got["dq"], got["dk"], got["dv"], **kw)
    else:
        width = -(-max(nk) // paged)
        order = torch.randperm(len(nk) * width, generator=torch.Generator().manual_seed(5)).view(len(nk), width)
        pages = [torch.full((len(nk) * width, paged, hk, dim), math.nan, dtype=d["k"].dtype, device="cuda") for _ in range(2)]
        for s, n in enumerate(nk):
            first = int(starts(nk)[s])
            at = torch.arange(n)
            rows = (order[s][at // paged] * paged + at % paged).cuda()
            for t, p in zip((d["k"], d["v"]), pages):
                p.flatten(0, 1)[rows] = t[first:first + n]
        op.paged_dev(d["q"], *pages, order.int().cuda(), cu_q, torch.tensor(nk, dtype=torch.int32, device="cuda"), got["out"],
                     got["lse"], max_q=max(nq), max_kv=max(nk))
    torch.cuda.synchronize()
    return got, op


def close(what, got, want, bound):
    import torch

    if not want.numel():
        return
    infinite = torch.isinf(want)
    assert torch.equal(got.double()[infinite], want[infinite]), what
    off = ((got.double() - want).abs() / (bound + 1e-7 * bound.max()))[~infinite]
    assert not len(off) or float(off.max()) <= 1.0, f"{what}: {float(off.max()):.3f} of the bound"


def compare(case, got, d):
    import torch

    import frame_attention_reference as ref

    name, dim, hq, hk, nq, nk, *window = case
    dtype, group, train = getattr(torch, TYPES[name]), hq // hk, "dq" in got
    cq, ck = starts(nq).tolist(), starts(nk).tolist()
    for s in range(len(nq)):
        rq, rk = slice(cq[s], cq[s + 1]), slice(ck[s], ck[s + 1])
        seen = visible(nq[s], nk[s], *window)
        for kh in range(hk):
            sums = {n: [0.0, 0.0] for n in ("dk", "dv")}
            for h in range(kh * group, (kh + 1) * group):
                want = ref.attention(d["q"][rq, h], d["k"][rk, kh], d["v"][rk, kh], seen, 1 / math.sqrt(dim), dtype,
                                     d["dout"][rq, h] if train else None)
                for n in ("out", "lse") + (("dq",) if train else ()):
                    close(f"{n} of sequence {s}, head {h}", got[n][rq, h], *want[n])
                for n in sums if train else ():
                    sums[n] = [a + b for a, b in zip(sums[n], want[n])]
            for n, (value, bound) in sums.items():
                if train:
                    close(f"{n} of sequence {s}, key head {kh}", got[n][rk, kh], value, bound)
    for n, t in got.items():  # rows of no sequence are as they were
        assert torch.isnan(t[:2]).all() and torch.isnan(t[-1:]).all(), n


def test_visible():
    import torch

    import frame_attention_reference as ref

    for case in ((20, 31, 1, 5, 0, 2), (31, 20, 4, 1, 1, 1), (9, 9, 3, -1, 0, 0), (7, 12, 2, 0, -1, 2), (5, 0, 1, 0, 0, 0)):
        assert torch.equal(visible(*case, device="cpu"), ref.visible(*case)), case


@pytest.mark.parametrize("case", CASES, ids=name_of)
def test_step(case, gpu_ctx):
    import torch

    print("case: step", case, flush=True)
    d = make(case, 1)
    got, _ = step(gpu_ctx, case, d)
    compare(case, got, d)
    again, _ = step(gpu_ctx, case, d)
    for n in got:
        assert torch.equal(got[n].nan_to_num(-7.0), again[n].nan_to_num(-7.0)), n


@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("case", CASES, ids=name_of)
def test_paged(case, page, gpu_ctx):
    print("case: paged", case, page, flush=True)
    d = make(case, 2)
    got, _ = step(gpu_ctx, case, d, page)
    compare(case, got, d)


@pytest.mark.parametrize("case,parts,sinks,sink_parts", PARTS, ids=[name_of(p[0]) for p in PARTS])
def test_key_gradients_in_parts(case, parts, sinks, sink_parts, gpu_ctx):
    import torch

    print("case: parts", case, flush=True)
    d = make(case, 3)
    got, op = step(gpu_ctx, case, d)
    compare(case, got, d)
    items = sinks * sink_parts + (-(-max(case[5]) // 128) - sinks) * (parts if parts > 1 else 0)
    deltas = (len(d["q"]) * case[2] + 3) // 4 * 4
    assert list(op._sizes.values())[-1] == 4 * (deltas + len(case[4]) * case[3] * items * 2 * 128 * case[1])
    again, _ = step(gpu_ctx, case, d)
    for n in got:
        assert torch.equal(got[n].nan_to_num(-7.0), again[n].nan_to_num(-7.0)), n
