"""FrameAttention outside the 16-bit heads of 64 and 128 channels: FP32, other head sizes and
tensors that are not aligned, forward, backward and paged, against the definition in 64 bits,
with infinities and NaN where nothing sees them. Bounds as in frame_attention_reference."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# dtype, head_dim, q_heads, kv_heads, queries, keys, frame, back, ahead, sinks, padding of a row
CASES = [
    ("f32", 64, 4, 2, 77, 77, 1, -1, 0, 0, 0),
    ("f32", 128, 2, 2, 65, 130, 5, 2, 0, 1, 0),
    ("f32", 33, 3, 1, 50, 61, 1, 9, 0, 3, 1),
    ("f32", 1, 2, 1, 40, 40, 1, -1, -1, 0, 0),
    ("f32", 200, 2, 1, 45, 70, 7, 1, 1, 1, 0),
    ("f16", 96, 6, 2, 70, 70, 4, 3, 0, 1, 0),
    ("bf16", 64, 4, 4, 66, 99, 1, 20, 0, 2, 3),  # rows off 16-byte alignment
    ("f16", 128, 8, 1, 33, 64, 16, 0, 0, 1, 1),
    ("bf16", 130, 2, 2, 34, 50, 1, -1, 0, 0, 0),
    ("f32", 64, 2, 1, 60, 20, 1, 4, 0, 0, 0),  # queries before the first key see nothing
]


def make(case, seed):
    name, dim, q_heads, kv_heads, nq, nk, frame, back, ahead, sinks, pad = case
    g = torch.Generator().manual_seed(seed)

    def heads(tokens, n):
        t = torch.randn(tokens, n, dim + pad, generator=g).to(TYPES[name])
        return t
    return [heads(nq, q_heads), heads(nk, kv_heads), heads(nk, kv_heads), heads(nq, q_heads)]


def run(ctx, case, q, k, v, dout):
    """(out, lse, dq, dk, dv) on the CPU; rows are views into padded ones."""
    from jasnamacos_amd.frame_attention import FrameAttention

    name, dim, q_heads, kv_heads, nq, nk, frame, back, ahead, sinks, pad = case
    op = FrameAttention(ctx, q_heads, kv_heads, dim, frame, back, ahead, sinks)
    tq, tk, tv, td = (t.cuda()[..., :dim] for t in (q, k, v, dout))
    out, dq = (torch.full((nq, q_heads, dim + pad), math.nan, dtype=TYPES[name], device="cuda")[..., :dim] for _ in range(2))
    dk, dv = (torch.full((nk, kv_heads, dim + pad), math.nan, dtype=TYPES[name], device="cuda")[..., :dim] for _ in range(2))
    lse = torch.empty(nq, q_heads, device="cuda")
    op.forward_dev(tq, tk, tv, out, lse, max_q=nq, max_kv=nk)
    op.backward_dev(tq, tk, tv, out, lse, td, dq, dk, dv, max_q=nq, max_kv=nk)
    return [t.cpu() for t in (out, lse, dq, dk, dv)]


def check(case, got, q, k, v, dout, seen):
    import frame_attention_reference as ref

    name, dim, q_heads, kv_heads = case[:4]
    group = q_heads // kv_heads
    want_k = {}
    for h in range(q_heads):
        kh = h // group
        want = ref.attention(q[:, h, :dim], k[:, kh, :dim], v[:, kh, :dim], seen, 1 / math.sqrt(dim), TYPES[name], dout[:, h, :dim])
        for key, t in (("out", got[0]), ("lse", got[1]), ("dq", got[2])):
            value, bound = want[key]
            mine = t[:, h].double()
            same = (mine == value) | ((mine - value).abs() <= bound)
            assert same.all(), f"{key} head {h}: {((mine - value).abs() / bound).nan_to_num(0).max()}"
        for key in ("dk", "dv"):
            a = want_k.setdefault((key, kh), [0, 0])
            a[0], a[1] = a[0] + want[key][0], a[1] + want[key][1]
    for (key, kh), (value, bound) in want_k.items():
        mine = got[3 if key == "dk" else 4][:, kh].double()
        assert ((mine - value).abs() <= bound).all(), f"{key} head {kh}: {((mine - value).abs() / bound).max()}"


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}-{c[1]}-{c[4]}x{c[5]}")
def test_against_the_definition(case, gpu_ctx):
    import frame_attention_reference as ref

    q, k, v, dout = make(case, 1)
    seen = ref.visible(case[4], case[5], *case[6:10])
    got = run(gpu_ctx, case, q, k, v, dout)
    check(case, got, q, k, v, dout, seen)
    again = run(gpu_ctx, case, q, k, v, dout)
    for a, b in zip(got, again):
        assert torch.equal(a.view(torch.int32 if a.element_size() == 4 else torch.int16),
                           b.view(torch.int32 if b.element_size() == 4 else torch.int16))


@pytest.mark.parametrize("case", [CASES[1], CASES[2], CASES[5], CASES[6], CASES[7]], ids=lambda c: f"{c[0]}-{c[1]}")
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_nothing_sees_reaches_nothing(case, value, gpu_ctx):
    """Rows of keys past a row's reach hold NaN and infinities: rows that do not see them are as with
    zeros there, bit for bit."""
    import frame_attention_reference as ref

    q, k, v, dout = make(case, 2)
    seen = ref.visible(case[4], case[5], *case[6:10])
    last = case[5] - 1
    rows = ~seen[:, last]
    assert rows.any()
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[last], clean_v[last] = 0, 0
    k[last], v[last] = value, value
    got, want = run(gpu_ctx, case, q, k, v, dout), run(gpu_ctx, case, q, clean_k, clean_v, dout)
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a[rows], b[rows])
    keys = seen[rows].any(0) & ~seen[~rows].any(0) if (~rows).any() else seen.any(0)
    for a, b in zip(got[3:], want[3:]):
        assert torch.equal(a[keys], b[keys])


@pytest.mark.parametrize("name,dim,page", [("f32", 64, 4), ("f32", 130, 1), ("f16", 96, 16), ("bf16", 64, 2)])
@pytest.mark.parametrize("new", [1, 5])
def test_paged(name, dim, page, new, gpu_ctx):
    """Ragged histories (one empty), pages in any order, NaN in pages' unused rows."""
    import frame_attention_reference as ref
    from jasnamacos_amd.frame_attention import FrameAttention

    dtype, q_heads, kv_heads = TYPES[name], 4, 2
    g = torch.Generator().manual_seed(3)
    lens = [0, new, 37, 64, 301]
    width = -(-max(lens) // page)
    table = torch.randperm(len(lens) * width, generator=g).view(len(lens), width).to(torch.int32)
    pages = [torch.full((len(lens) * width, page, kv_heads, dim), math.nan, dtype=dtype) for _ in range(2)]
    q = torch.randn(len(lens) * new, q_heads, dim, generator=g).to(dtype)
    rows = []
    for s, n in enumerate(lens):
        kv = [torch.randn(n, kv_heads, dim, generator=g).to(dtype) for _ in range(2)]
        rows.append(kv)
        for j in range(n):
            for t, p in zip(kv, pages):
                p[table[s, j // page], j % page] = t[j]
    op = FrameAttention(gpu_ctx, q_heads, kv_heads, dim, back=40, sinks=3)
    out = torch.empty_like(q, device="cuda")
    lse = torch.empty(len(q), q_heads, device="cuda")
    op.paged_dev(q.cuda(), pages[0].cuda(), pages[1].cuda(), table.cuda(), None,
                 torch.tensor(lens, dtype=torch.int32, device="cuda"), out, lse, max_q=new)
    for s, n in enumerate(lens):
        run_ = slice(s * new, (s + 1) * new)
        seen = ref.visible(new, n, 1, 40, 0, 3)
        for h in range(q_heads):
            want = ref.attention(q[run_, h], rows[s][0][:, h // 2], rows[s][1][:, h // 2], seen, 1 / math.sqrt(dim), dtype)
            for key, t in (("out", out), ("lse", lse)):
                value, bound = want[key]
                mine = t[run_, h].double().cpu()
                assert ((mine == value) | ((mine - value).abs() <= bound)).all(), (key, s, h)
