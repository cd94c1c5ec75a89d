"""Workloads that the speed of the operators of a microscaled cache and of shared prefixes is
measured on (jasnamacos_amd.frame_attention), and their plain forms in torch.

The tokens are patches of the framework's maps: a 64 x 64 tile is 16 x 16 or 8 x 8 tokens a
frame, the 180 x 320 map 45 x 80; clips have up to 30 frames. Heads have 64 channels, as the
framework's features do, or 128.

A microscaled cache keeps blocks of 32 channels as codes of 8 bits (e4m3) or 4 (e2m1) and one
power of two; a head's tokens of a page lie together: codes [pages][kv_heads][page][dim] (4 bits:
two channels a byte, the first one low), scales [pages][kv_heads][page][dim / 32] (exponent + 127).

Every case is a dict: "kind" says which operator, the rest its sizes.
  append  CacheAppend.run_mx_dev: rotated keys and values into microscaled pages, queries rotated on the way
  read    CacheRead.run_dev: what a microscaled cache holds of the last tokens, in 16 or 32 bits
  attend  FrameAttention.paged_mx_dev: new tokens against a microscaled cache
  shared  FrameAttention.shared_dev: new tokens of streams that share a prefix, whose own tokens
          come after it; "bits" 16: pages of the tensors' type, else microscaled
"""
import math

import numpy as np
import torch

own = False

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_LARGEST = {8: 448.0, 4: 6.0}  # of e4m3 and e2m1
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- the cases -------------------------------------------------------------------------

def listed():
    return [
        # One new token of each of 48 streams that are served together.
        {"name": "append_token_f16", "kind": "append", "dtype": "f16", "sequences": 48, "new": 1, "longest": 700, "page": 16,
         "q_heads": 16, "kv_heads": 4, "dim": 128},
        # A whole new frame of the 180 x 320 map for each of 8 streams.
        {"name": "append_frame_bf16", "kind": "append", "dtype": "bf16", "sequences": 8, "new": 3600, "longest": 14400, "page": 64,
         "q_heads": 8, "kv_heads": 8, "dim": 64},
        # The last frame of one stream of a tile, out of a 4-bit cache.
        {"name": "read_frame_f16", "kind": "read", "dtype": "f16", "bits": 4, "sequences": 1, "new": 256, "longest": 777, "page": 16,
         "kv_heads": 4, "dim": 64},
        # The histories of four streams of the 180 x 320 map, to move them to a cache of 16 bits.
        {"name": "read_clip_bf16", "kind": "read", "dtype": "bf16", "bits": 8, "sequences": 4, "new": 14400, "longest": 36000,
         "page": 64, "kv_heads": 8, "dim": 128},
        # One stream, one token: the smallest call of serving.
        {"name": "attend_token_f16", "kind": "attend", "dtype": "f16", "bits": 8, "sequences": 1, "new": 1, "longest": 997, "page": 16,
         "q_heads": 8, "kv_heads": 8, "dim": 64, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        # 32 streams with long histories, one token each, in 8 bits and in 4.
        {"name": "attend_batch_bf16", "kind": "attend", "dtype": "bf16", "bits": 8, "sequences": 32, "new": 1, "longest": 18001,
         "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        {"name": "attend_batch_4bit_f16", "kind": "attend", "dtype": "f16", "bits": 4, "sequences": 32, "new": 1, "longest": 18001,
         "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        # A frame of the 180 x 320 map for each of two streams, the last three frames and the first one visible.
        {"name": "attend_frame_bf16", "kind": "attend", "dtype": "bf16", "bits": 8, "sequences": 2, "new": 3600, "longest": 14400,
         "page": 64, "q_heads": 8, "kv_heads": 8, "dim": 64, "frame": 3600, "back": 2, "ahead": 0, "sinks": 1},
        # Four continuations of one tile's clip, one token each.
        {"name": "shared_token_f16", "kind": "shared", "dtype": "f16", "bits": 16, "sequences": 4, "new": 1, "prefix": 1024,
         "longest": 41, "page": 16, "q_heads": 8, "kv_heads": 8, "dim": 64, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        # 64 continuations of four frames of the 180 x 320 map, one token each, in 16 bits and in 8.
        {"name": "shared_batch_bf16", "kind": "shared", "dtype": "bf16", "bits": 16, "sequences": 64, "new": 1, "prefix": 14400,
         "longest": 901, "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        {"name": "shared_batch_8bit_bf16", "kind": "shared", "dtype": "bf16", "bits": 8, "sequences": 64, "new": 1, "prefix": 14400,
         "longest": 901, "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        # Eight continuations of a 30-frame clip of a tile, a whole frame each, half the clip and its first frame visible.
        {"name": "shared_frame_f16", "kind": "shared", "dtype": "f16", "bits": 16, "sequences": 8, "new": 256, "prefix": 7680,
         "longest": 768, "page": 64, "q_heads": 8, "kv_heads": 4, "dim": 64, "frame": 256, "back": 15, "ahead": 0, "sinks": 1},
    ]


def _log(rng, low, high):
    """A whole number spread over low..high by its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "attend", "shared", "shared", "shared"])
    case = {"kind": kind, "dtype": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128]), "dim": rng.choice([64, 128])}
    kv = rng.choice([1, 2, 4, 8])
    q = kv * rng.choice([g for g in (1, 2, 3, 4, 8) if kv * g <= 32])
    dim = case["dim"]
    if kind in ("append", "read"):
        case["dtype"] = rng.choice(["f16", "bf16", "f32"])
        case["dim"] = dim = rng.choice([64, 128, 32, 96])
        sequences = rng.randint(1, 64)
        each = sequences * (q + 2 * kv if kind == "append" else 2 * kv) * dim
        new = _log(rng, 1, max(1, min(3600, 28800 * 24 * 64 // each)))
        case.update(sequences=sequences, new=new, longest=new + _log(rng, 1, 2 * new + 500), kv_heads=kv)
        case.update({"q_heads": q} if kind == "append" else {"bits": rng.choice([8, 4])})
        return case
    frame = rng.choice([1, 1, 64, 256, rng.randint(2, 300)])
    sequences = rng.randint(1, 32) if kind == "attend" else rng.randint(2, 64)
    case.update(bits=rng.choice([8, 8, 4] if kind == "attend" else [16, 16, 8, 4]), sequences=sequences, q_heads=q, kv_heads=kv,
                frame=frame, ahead=0, sinks=rng.choice([0, 1, 4]))
    if kind == "shared":
        case["prefix"] = _log(rng, 64, 14400)
        longest = _log(rng, 1, min(2000, 64 * 901 * 8 * 128 // (sequences * kv * dim)))
    else:
        longest = _log(rng, 100, min(18001, 32 * 18001 * 8 * 128 // (sequences * kv * dim)))
    keys = longest + case.get("prefix", 0)
    new = rng.choice([1, 1, min(frame, longest), rng.randint(1, 16)])
    case["new"] = max(1, min(new, longest, 2048 // sequences, int(1e11 / (4 * dim * q * keys * sequences))))
    case["longest"] = longest
    case["back"] = rng.choice([-1, max(1, keys // (2 * frame))])
    return case


# ---- inputs ----------------------------------------------------------------------------

def _lengths(case):
    """The sequences' own lengths: the longest first, the others spread over a third of it and more."""
    share = [1.0 if i == 0 else 0.35 + 0.65 * ((i * 0.618) % 1.0) for i in range(case["sequences"])]
    return [max(case["new"], int(case["longest"] * s)) for s in share]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class _Random:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(int(seed))

    def normal(self, *size, dtype=torch.float32):
        return torch.randn(size, generator=self.gen, device="cuda").to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda").to(torch.int32)


def _sections(dim):
    """How many of a head's pairs turn with the time, the height and the width."""
    side = 3 * (dim // 2) // 8
    return dim // 2 - 2 * side, side, side


def _frequencies(dim):
    """The angle a step of each pair: each axis starts at 1 and falls to 1 / 1000."""
    parts = [1000.0 ** (-torch.arange(n, dtype=torch.float64) / max(1, n)) for n in _sections(dim)]
    return torch.cat(parts).float().cuda()


def _grid(first, tokens):
    """[tokens][3]: (time, height, width) of the tokens first, first + 1, ... of 45 x 80 frames."""
    n = torch.arange(tokens, device="cuda", dtype=torch.int64) + first
    return torch.stack([n // 3600, n // 80 % 45, n % 80], 1).to(torch.int32).contiguous()


def _pool(r, pages, case):
    """The buffers of a cache with this many pages, as a stream that has run would have left them."""
    page, heads, dim, bits = case["page"], case["kv_heads"], case["dim"], case.get("bits", 8)
    if bits == 16:
        return [r.normal(pages, page, heads, dim, dtype=_DTYPE[case["dtype"]]) for _ in range(2)]
    codes, scales = [], []
    for _ in range(2):
        done = [_quantised(r.normal(len(n), heads, page, dim), bits) for n in torch.arange(pages).split(1 + (1 << 27) // (heads * page * dim))]
        codes.append(torch.cat([_packed(c, bits) for c, _ in done]))
        scales.append(torch.cat([(e + 127).to(torch.uint8) for _, e in done]))
    return codes + scales


def prepare(case, seed):
    """Queries, keys and values ~ N(0, 1), as after a norm; pages in a random order, with a few to spare."""
    r = _Random(seed)
    kind, dtype = case["kind"], _DTYPE[case["dtype"]]
    lengths, b, new, page = _lengths(case), case["sequences"], case["new"], case["page"]
    prefix = case.get("prefix", 0)
    used = [-(-n // page) for n in [prefix] + lengths]
    order = r.order(sum(used) + 3)
    table = torch.full((b, max(used[1:])), -1, dtype=torch.int32, device="cuda")
    at = used[0]
    for row, n in zip(table, used[1:]):
        row[:n] = order[at:at + n]
        at += n
    s = {"case": case, "lengths": lengths, "table": table, "kv_lens": _ints(lengths), "cu": _ints([i * new for i in range(b + 1)]),
         "pool": _pool(r, sum(used) + 3, case)}
    hk, d = case["kv_heads"], case["dim"]
    if kind == "read":
        s["k_out"], s["v_out"] = (torch.empty(b * new, hk, d, dtype=dtype, device="cuda") for _ in range(2))
        return s
    hq = case["q_heads"]
    packed = r.normal(b * new, hq + 2 * hk, d, dtype=dtype)
    s["q"], s["out"] = packed[:, :hq], torch.empty(b * new, hq, d, dtype=dtype, device="cuda")
    if kind == "append":
        s["k"], s["v"] = packed[:, hq:hq + hk], packed[:, hq + hk:]
        s["positions"] = torch.cat([_grid(n - new, new) for n in lengths])
        s["freq"] = _frequencies(d)
    if kind == "shared":
        s["prefix_table"], s["prefix_len"] = order[:used[0]].clone(), _ints([prefix])
    return s


# ---- one pass through the framework's operators ------------------------------------------

_KEEP = {}


def _handle(name, *sizes):
    """The handles that a program keeps: one context, and one of each operator it has."""
    from jasnamacos_amd import deform_conv as dc
    from jasnamacos_amd import frame_attention as fa

    if "ctx" not in _KEEP:
        _KEEP["ctx"] = dc.HipDeformConv(0)
    key = (name,) + sizes
    if key not in _KEEP:
        _KEEP[key] = getattr(fa, name)(_KEEP["ctx"], *sizes)
    return _KEEP[key]


def _pages(s):
    """The cache as the calls take it: kept with its buffers."""
    if "pages" not in s:
        from jasnamacos_amd import frame_attention as fa

        s["pages"] = tuple(s["pool"]) if len(s["pool"]) == 2 else fa.MxPages(*s["pool"])
    return s["pages"]


def _run_own(s):
    case, pages = s["case"], _pages(s)
    kind = case["kind"]
    if kind == "append":
        turn = _handle("Rotary", case["dim"], _sections(case["dim"]), False)
        _handle("CacheAppend").run_mx_dev(s["k"], s["v"], pages, s["table"], s["cu"], s["kv_lens"], rotary=turn,
                                          positions=s["positions"], freq=s["freq"], q=s["q"], q_out=s["out"])
        return _kept(s)
    if kind == "read":
        _handle("CacheRead").run_dev(pages, s["table"], s["cu"], s["kv_lens"], s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"]}
    op = _handle("FrameAttention", case["q_heads"], case["kv_heads"], case["dim"], case["frame"], case["back"], case["ahead"],
                 case["sinks"])
    if kind == "attend":
        op.paged_mx_dev(s["q"], pages, s["table"], s["cu"], s["kv_lens"], s["out"], max_q=case["new"], max_kv=s["lengths"][0])
    else:
        op.shared_dev(s["q"], pages, s["prefix_table"], s["prefix_len"], s["table"], s["cu"], s["kv_lens"], s["out"],
                      max_q=case["new"], max_kv=s["lengths"][0], max_prefix=case["prefix"])
    return s["out"]


def _kept(s):
    """What an append leaves: the queries, and the cache's buffers as the numbers that their bytes are."""
    k, v, ks, vs = s["pool"]
    return {"q": s["out"], "k": k.view(torch.float8_e4m3fn), "v": v.view(torch.float8_e4m3fn),
            "k_scales": ks.view(torch.float8_e8m0fnu), "v_scales": vs.view(torch.float8_e8m0fnu)}


# ---- the plain forms ---------------------------------------------------------------------

def _quantised(x, bits):
    """(codes as numbers, exponents of their blocks) of x [...][dim] in 32 bits: the smallest power of
    two that takes a block's largest magnitude to what a code can hold, codes to the nearest, ties to even."""
    blocks = x.unflatten(-1, (-1, 32))
    share, e = torch.frexp(blocks.abs().amax(-1) / _LARGEST[bits])  # share in [0.5, 1)
    e = torch.where(share == 0.5, e - 1, torch.where(share == 0, -127, e)).clamp(min=-127)
    scaled = torch.ldexp(blocks, -e[..., None])
    if bits == 8:
        codes = scaled.to(torch.float8_e4m3fn).float()
    else:  # steps of 0.5 up to 2, of 1 up to 4, of 2 above
        size = scaled.abs()
        step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
        codes = torch.copysign(torch.round(size / step) * step, scaled)
    return codes.flatten(-2), e


def _packed(codes, bits):
    """Codes as bytes: e4m3, or two e2m1 a byte."""
    if bits == 8:
        return codes.to(torch.float8_e4m3fn).view(torch.uint8)
    size = codes.abs()
    index = torch.where(size < 2, 2 * size, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    index = (index + 8 * torch.signbit(codes)).to(torch.uint8)
    return index[..., 0::2] | (index[..., 1::2] << 4)


def _values(codes, scales, bits):
    """[...][dim] in 32 bits of what bytes of codes and scales hold."""
    if bits == 8:
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        two = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
        x = torch.tensor(_E2M1, device=codes.device)[(two & 7).long()] * (1.0 - 2.0 * (two >> 3).float())
    return torch.ldexp(x.unflatten(-1, (-1, 32)), (scales.int() - 127)[..., None]).flatten(-2)


def _turned(x, positions, freq):
    """x [tokens][heads][dim] in 32 bits, channel i turned with channel i + dim / 2; the angles in 64 bits."""
    pairs = freq.numel()
    st, sh, _ = _sections(2 * pairs)
    pair = torch.arange(pairs, device=x.device)
    axis = (pair >= st).long() + (pair >= st + sh).long()
    angle = torch.remainder(positions[:, axis].double() * freq.double(), 2 * math.pi)[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :pairs], x[..., pairs:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _places(s):
    """(page, token of the page) of each of the new tokens, in order."""
    case = s["case"]
    at = (s["kv_lens"].long()[:, None] - case["new"] + torch.arange(case["new"], device="cuda")).reshape(-1)
    row = torch.arange(case["sequences"], device="cuda").repeat_interleave(case["new"])
    return s["table"][row, at // case["page"]].long(), at % case["page"]


def _gathered(s, table, most):
    """Keys and values of the tables' first `most` tokens: [sequences][heads][most][dim] in 32 bits."""
    case, pool = s["case"], s["pool"]
    which = table.clamp(min=0).long()
    got = []
    for n in range(2):
        if case["bits"] == 16:
            x = pool[n][which].float().transpose(2, 3)
        else:
            x = _values(pool[n][which], pool[n + 2][which], case["bits"])
        got.append(x.transpose(1, 2).flatten(2, 3)[:, :, :most].contiguous())
    return got


def _visible(p, keys, case):
    """Which keys (their places) queries at places p [sequences][queries] see."""
    f = case["frame"]
    fp, fj = torch.div(p, f, rounding_mode="floor")[..., None], torch.div(keys, f, rounding_mode="floor")
    seen = torch.ones_like(fp, dtype=torch.bool) & (fj >= 0)
    if case["ahead"] >= 0:
        seen = seen & (fj <= fp + case["ahead"])
    if case["back"] >= 0:
        seen = seen & ((fj >= fp - case["back"]) | (fj < case["sinks"]))
    return seen


def _attended(s):
    """Attention of the new tokens over the prefix, if there is one, and their own tokens."""
    case = s["case"]
    b, new, hq, hk, d = (case[n] for n in ("sequences", "new", "q_heads", "kv_heads", "dim"))
    group, prefix, most = hq // hk, case.get("prefix", 0), s["lengths"][0]
    q = s["q"].float().reshape(b, new, hk, group, d)
    own_len = s["kv_lens"].long()
    p = prefix + own_len[:, None] - new + torch.arange(new, device="cuda")
    j = torch.arange(most, device="cuda")
    k, v = _gathered(s, s["table"], most)
    by_own = q.permute(0, 2, 3, 1, 4).reshape(b, hk, group * new, d)
    scores = torch.matmul(by_own, k.transpose(2, 3)).reshape(b, hk, group, new, most) * (1.0 / math.sqrt(d))
    seen = _visible(p, prefix + j, case) & (j < own_len[:, None])[:, None]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    if prefix:
        kp, vp = (x[0] for x in _gathered(s, s["prefix_table"][None], prefix))
        by_prefix = q.permute(2, 0, 3, 1, 4).reshape(hk, b * group * new, d)
        first = torch.matmul(by_prefix, kp.transpose(1, 2)) * (1.0 / math.sqrt(d))
        first = first.reshape(hk, b, group, new, prefix).transpose(0, 1)
        first = first.masked_fill(~_visible(p, torch.arange(prefix, device="cuda"), case)[:, None, None], -math.inf)
        scores = torch.cat([first, scores], -1)
        del first
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(e[..., prefix:].reshape(b, hk, group * new, most), v).reshape(b, hk, group, new, d)
    if prefix:
        first = e[..., :prefix].transpose(0, 1).reshape(hk, b * group * new, prefix)
        out = out + torch.matmul(first, vp).reshape(hk, b, group, new, d).transpose(0, 1)
    return out.permute(0, 3, 1, 2, 4).reshape(b * new, hq, d).to(_DTYPE[case["dtype"]])


def _run_plain(s):
    case = s["case"]
    kind, dtype = case["kind"], _DTYPE[case["dtype"]]
    if kind in ("attend", "shared"):
        return _attended(s)
    which, at = _places(s)
    if kind == "read":
        k, v = (_values(s["pool"][n][which, :, at], s["pool"][n + 2][which, :, at], case["bits"]).to(dtype) for n in range(2))
        return {"k": k, "v": v}
    s["out"].copy_(_turned(s["q"].float(), s["positions"], s["freq"]))
    for n, x in enumerate((_turned(s["k"].float(), s["positions"], s["freq"]), s["v"].float())):
        codes, e = _quantised(x, 8)
        s["pool"][n][which, :, at] = _packed(codes, 8)
        s["pool"][n + 2][which, :, at] = (e + 127).to(torch.uint8)
    return _kept(s)


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- what a pass cannot do without ---------------------------------------------------------

def _seen(case):
    """(visible pairs of query and key, own keys that any query sees, keys of the prefix that any sees)."""
    prefix, f = case.get("prefix", 0), case["frame"]
    pairs, keys, first = 0, 0, (prefix, 0, 0)  # the prefix: from, to, sinks
    for n in _lengths(case):
        p = np.arange(prefix + n - case["new"], prefix + n, dtype=np.int64)
        high = np.full_like(p, prefix + n) if case["ahead"] < 0 else np.minimum(prefix + n, (p // f + case["ahead"] + 1) * f)
        low = np.zeros_like(p) if case["back"] < 0 else np.minimum(high, np.maximum(0, (p // f - case["back"]) * f))
        sinks = np.minimum(case["sinks"] * f, low)
        pairs += int((high - low + sinks).sum())
        a, b, c = int(low.min()), int(high.max()), int(sinks.max())
        keys += max(0, b - max(a, prefix)) + max(0, min(c, a) - prefix)
        first = (min(first[0], a), max(first[1], min(b, prefix)), max(first[2], min(c, prefix)))
    return pairs, keys, max(0, first[1] - first[0]) + min(first[2], first[0])


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kind, hk, d = case["kind"], case["kv_heads"], case["dim"]
    each = d * size if case.get("bits", 8) == 16 else d * case.get("bits", 8) // 8 + d // 32  # bytes of a key
    tokens = case["sequences"] * case["new"]
    if kind == "read":
        return {"bytes": tokens * 2 * hk * (each + d * size), "flops": tokens * 2 * hk * d}
    hq = case["q_heads"]
    if kind == "append":
        return {"bytes": tokens * ((2 * hq + 2 * hk) * d * size + 2 * hk * each + 12),
                "flops": tokens * ((hq + hk) * d // 2 * 6 + 4 * hk * d)}
    pairs, keys, first = _seen(case)
    return {"bytes": 2 * tokens * hq * d * size + 2 * (keys + first) * hk * each, "flops": 4 * d * hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------

def _exact_values(codes, scales, bits):
    """A code's number from its fields: sign, exponent (bias 7 or 1), fraction (3 bits or 1)."""
    scale = torch.pow(2.0, scales.double() - 127.0)
    if bits == 4:
        codes = torch.stack([codes % 16, codes // 16], -1).reshape(*codes.shape[:-1], -1)
    width, bias, fraction = (4, 7, 3) if bits == 8 else (2, 1, 1)
    c = codes.long()
    exponent, rest = (c >> fraction) % (1 << width), (c % (1 << fraction)).double() / (1 << fraction)
    size = torch.where(exponent > 0, (1.0 + rest) * torch.pow(2.0, exponent.double() - bias), rest * 2.0 ** (1 - bias))
    signed = torch.where((c >> (fraction + width)) > 0, -size, size)
    return (signed.reshape(*scale.shape, 32) * scale[..., None]).reshape(signed.shape)


def _exact_turn(x, positions, freq):
    n = freq.numel()
    angle = torch.cat([positions[:, a:a + 1].double() * f for a, f in enumerate(torch.split(freq.double(), list(_sections(2 * n))))], 1)
    z = torch.complex(x[..., :n].double(), x[..., n:].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_rows(s, table, n, part):
    """[n][heads][dim]: the first n tokens of one table in 64 bits; part 0: keys, 1: values."""
    case, pool = s["case"], s["pool"]
    pages = table[:-(-n // case["page"])].long()
    if case.get("bits", 8) == 16:
        return pool[part][pages].double().flatten(0, 1)[:n]
    x = _exact_values(pool[part][pages], pool[part + 2][pages], case["bits"])
    return x.transpose(1, 2).flatten(0, 1)[:n]


def exact(case, seed):
    """For an append: the codes before they are rounded to 8 bits (blocks that it does not write as they
    were), which says how much the rounding takes; the scales are whole powers of two."""
    s = prepare(case, seed)
    kind, new, page = case["kind"], case["new"], case["page"]
    if kind == "read":
        got = [torch.cat([_exact_rows(s, s["table"][b], n, part)[n - new:] for b, n in enumerate(s["lengths"])]) for part in range(2)]
        return {"k": got[0], "v": got[1]}
    if kind == "append":
        got = {"q": _exact_turn(s["q"], s["positions"], s["freq"])}
        for name, x, codes, scales in (("k", _exact_turn(s["k"], s["positions"], s["freq"]), s["pool"][0], s["pool"][2]),
                                       ("v", s["v"].double(), s["pool"][1], s["pool"][3])):
            every = _exact_values(codes, torch.full_like(scales, 127), 8)
            exponents = scales.double() - 127.0
            for b, n in enumerate(s["lengths"]):
                at = torch.arange(n - new, n, device="cuda")
                which, at = s["table"][b].long()[at // page], at % page
                rows = x[b * new:(b + 1) * new]
                blocks = rows.reshape(*rows.shape[:-1], -1, 32)
                e = torch.ceil(torch.log2(blocks.abs().amax(-1) / 448.0)).clamp(min=-127.0)
                every[which, :, at] = (blocks / torch.pow(2.0, e)[..., None]).reshape(rows.shape)
                exponents[which, :, at] = e
            got[name], got[name + "_scales"] = every, torch.pow(2.0, exponents)
        return got
    hq, prefix, f = case["q_heads"], case.get("prefix", 0), case["frame"]
    group = hq // case["kv_heads"]
    out = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda")
    before = [_exact_rows(s, s["prefix_table"], prefix, part) for part in range(2)] if prefix else None
    for b, n in enumerate(s["lengths"]):
        keys, values = (_exact_rows(s, s["table"][b], n, part) for part in range(2))
        if prefix:
            keys, values = torch.cat([before[0], keys]), torch.cat([before[1], values])
        place = torch.arange(prefix + n - new, prefix + n, device="cuda")[:, None]
        start = place - place % f  # the first token of the query's frame
        j = torch.arange(prefix + n, device="cuda")[None]
        mask = torch.ones(new, prefix + n, dtype=torch.bool, device="cuda")
        if case["ahead"] >= 0:
            mask &= j < start + (case["ahead"] + 1) * f
        if case["back"] >= 0:
            mask &= (j >= start - case["back"] * f) | (j < case["sinks"] * f)
        rows = slice(b * new, (b + 1) * new)
        for head in range(hq):
            scores = s["q"][rows, head].double() @ keys[:, head // group].T / math.sqrt(case["dim"])
            out[rows, head] = torch.softmax(scores.masked_fill(~mask, -math.inf), 1) @ values[:, head // group]
    return out
