"""Workloads that the speed of the frame-attention operators is measured on
(jasnamacos_amd.frame_attention), and their plain forms in torch.

The tokens are patches of the framework's maps: a 64 x 64 tile is 16 x 16 or 8 x 8 tokens a
frame, the 180 x 320 map 45 x 80; clips have up to 30 frames. Heads have 64 channels, as the
framework's features do, or 128.

Every case is a dict: "kind" says which operator, the rest its sizes.
  rotary  Rotary.run_dev: time, height and width rotations of packed queries and keys
  append  CacheAppend.run_dev: rotated keys and values into pages, queries rotated on the way
  attend  FrameAttention.forward_dev over whole sequences
  train   FrameAttention.forward_dev and backward_dev: a training step's attention
  paged   FrameAttention.paged_dev: new tokens against the paged cache
  norm    GatedNorm.forward_dev, and with "step" its backward_dev too
"""
import math

import numpy as np
import torch

own = False

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-6


# ---- the cases -------------------------------------------------------------------------

def listed():
    return [
        # The queries and keys of one frame of a tile in an FP32 model: launch and latency.
        {"name": "rotary_frame_f32", "kind": "rotary", "dtype": "f32", "frames": 1, "rows": 8, "columns": 8, "heads": 8,
         "others": 4, "dim": 64, "pairs": 32, "interleaved": False, "inverse": False},
        # The gradients of a 30-frame clip's queries and keys over the 180 x 320 map, back through the rotation.
        {"name": "rotary_clip_bf16", "kind": "rotary", "dtype": "bf16", "frames": 30, "rows": 45, "columns": 80,
         "heads": 16, "others": 8, "dim": 64, "pairs": 32, "interleaved": True, "inverse": True},
        # One new token of each of 64 streams that are served together.
        {"name": "append_token_f16", "kind": "append", "dtype": "f16", "sequences": 64, "new": 1, "longest": 511,
         "page": 16, "q_heads": 16, "kv_heads": 4, "dim": 128},
        # A whole new frame of the 180 x 320 map for each of 8 streams.
        {"name": "append_frame_bf16", "kind": "append", "dtype": "bf16", "sequences": 8, "new": 3600, "longest": 10800,
         "page": 64, "q_heads": 8, "kv_heads": 8, "dim": 64},
        # A few short sequences of odd lengths, causal by tokens.
        {"name": "attend_ragged_f16", "kind": "attend", "dtype": "f16", "sequences": 5, "longest": 301, "ragged": True,
         "q_heads": 8, "kv_heads": 8, "dim": 64, "frame": 1, "back": 127, "ahead": 0, "sinks": 4},
        # A 30-frame clip of a 64 x 64 tile, the last eight frames and the first one visible.
        {"name": "attend_clip_bf16", "kind": "attend", "dtype": "bf16", "sequences": 1, "longest": 7680, "ragged": False,
         "q_heads": 16, "kv_heads": 4, "dim": 128, "frame": 256, "back": 7, "ahead": 0, "sinks": 1},
        # Training on ragged sequences with shared key heads.
        {"name": "train_ragged_f16", "kind": "train", "dtype": "f16", "sequences": 4, "longest": 1021, "ragged": True,
         "q_heads": 8, "kv_heads": 2, "dim": 128, "frame": 1, "back": 255, "ahead": 0, "sinks": 4},
        # Training on four ten-frame windows of 16 x 16 tokens a frame.
        {"name": "train_clip_bf16", "kind": "train", "dtype": "bf16", "sequences": 4, "longest": 2560, "ragged": False,
         "q_heads": 8, "kv_heads": 8, "dim": 64, "frame": 256, "back": 3, "ahead": 0, "sinks": 1},
        # One stream, one token: the smallest call of serving.
        {"name": "decode_stream_f16", "kind": "paged", "dtype": "f16", "sequences": 1, "new": 1, "longest": 777,
         "page": 16, "q_heads": 8, "kv_heads": 8, "dim": 64, "frame": 1, "back": -1, "ahead": 0, "sinks": 0},
        # 32 streams with long histories, one token each.
        {"name": "decode_batch_bf16", "kind": "paged", "dtype": "bf16", "sequences": 32, "new": 1, "longest": 20011,
         "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "frame": 1, "back": 16383, "ahead": 0, "sinks": 64},
        # The norms around a block for one frame of a tile in an FP32 model.
        {"name": "norm_frame_f32", "kind": "norm", "dtype": "f32", "tokens": 64, "channels": 512, "gate_tokens": 64,
         "step": False},
        # A training step of the norms around a block: a 10-frame clip of the 180 x 320 map, a gate for each frame.
        {"name": "norm_clip_bf16", "kind": "norm", "dtype": "bf16", "tokens": 36000, "channels": 512, "gate_tokens": 3600,
         "step": True},
    ]


def _log(rng, low, high):
    """A whole number spread over low..high by its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([g for g in (1, 2, 3, 4, 8) if kv * g <= 32]), kv


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "train", "train", "paged", "paged", "norm"])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128])
    if kind == "rotary":
        heads = rng.randint(1, 24)
        tokens = _log(rng, 16, min(108000, 108000 * 16 * 64 // (heads * dim)))
        rows = rng.randint(1, max(1, min(45, tokens)))
        columns = rng.randint(1, max(1, min(80, tokens // rows)))
        return {"kind": kind, "dtype": rng.choice(["f16", "bf16", "f32"]), "frames": max(1, min(400, tokens // (rows * columns))),
                "rows": rows, "columns": columns, "heads": heads, "others": rng.randint(0, 8), "dim": dim,
                "pairs": rng.choice([dim // 2, dim // 2, dim // 4 + 3]), "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.5}
    if kind == "norm":
        channels = rng.choice([64, 256, 512, 1000, 1024, rng.randint(33, 2048)])
        groups = rng.randint(1, 30)
        gate = _log(rng, 1, max(1, 36000 * 512 // (channels * groups)))
        return {"kind": kind, "dtype": rng.choice(["f16", "bf16", "f32"]), "tokens": gate * groups, "channels": channels,
                "gate_tokens": gate, "step": rng.random() < 0.6}
    q_heads, kv_heads = _heads(rng)
    if kind == "append":
        sequences = rng.randint(1, 64)
        new = _log(rng, 1, max(1, min(3600, 28800 * 24 * 64 // (sequences * (q_heads + 2 * kv_heads) * dim))))
        return {"kind": kind, "dtype": dtype, "sequences": sequences, "new": new, "longest": new + _log(rng, 1, 2 * new + 500),
                "page": rng.choice([16, 32, 64, 128]), "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim}
    frame = rng.choice([1, 1, 64, 256, rng.randint(2, 300)])
    if kind == "paged":
        sequences = rng.randint(1, 32)
        longest = _log(rng, 100, min(20011, 32 * 20011 * 8 * 128 // (sequences * kv_heads * dim)))
        new = rng.choice([1, 1, min(frame, longest), rng.randint(1, 16)])
        new = max(1, min(new, longest, 2048 // sequences, int(1.1e11 / (4 * dim * q_heads * longest * sequences))))
        back = rng.choice([-1, max(1, longest // (2 * frame))])
        return {"kind": kind, "dtype": dtype, "sequences": sequences, "new": new, "longest": longest,
                "page": rng.choice([16, 32, 64, 128]), "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "frame": frame,
                "back": back, "ahead": 0, "sinks": rng.choice([0, 1, 4])}
    sequences = rng.randint(1, 6)
    most = math.sqrt(1.1e11 / ((4 if kind == "attend" else 14) * dim * q_heads * sequences))  # every pair visible
    longest = min(_log(rng, 64, 6000), int(most))
    return {"kind": kind, "dtype": dtype, "sequences": sequences, "longest": longest, "ragged": rng.random() < 0.6,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "frame": frame,
            "back": rng.choice([-1, max(1, longest // (3 * frame)), max(1, longest // (8 * frame))]),
            "ahead": rng.choice([0, 0, 0, 1, -1]), "sinks": rng.choice([0, 1, 4])}


# ---- inputs ----------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths: the longest first, the others spread over a third of it and more."""
    share = [1.0 if i == 0 or not case.get("ragged", True) else 0.35 + 0.65 * ((i * 0.618) % 1.0)
             for i in range(case["sequences"])]
    return [max(case.get("new", 1), int(case["longest"] * s)) for s in share]


def _starts(lengths):
    return [0] + [int(v) for v in np.cumsum(lengths)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class _Random:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(int(seed))

    def normal(self, *size, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(size, generator=self.gen, device="cuda") * std + mean).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda").to(torch.int32)


def _sections(pairs):
    """How many of the pairs turn with the time, the height and the width."""
    return pairs - 2 * (3 * pairs // 8), 3 * pairs // 8, 3 * pairs // 8


def _frequencies(pairs):
    """The angle a step of each pair: each axis starts at 1 and falls to 1 / 1000."""
    parts = [1000.0 ** (-torch.arange(n, dtype=torch.float64) / max(1, n)) for n in _sections(pairs)]
    return torch.cat(parts).float().cuda()


def _grid(first, tokens, rows, columns):
    """[tokens][3]: (time, height, width) of the tokens first, first + 1, ... in raster order."""
    n = torch.arange(tokens, device="cuda", dtype=torch.int64) + first
    return torch.stack([n // (rows * columns), n // columns % rows, n % columns], 1).to(torch.int32).contiguous()


def _pages(r, case):
    """A pool of pages with a few to spare, and each sequence's table of pages in a random order."""
    lengths = _lengths(case)
    width = -(-max(lengths) // case["page"])
    used = [-(-n // case["page"]) for n in lengths]
    order = r.order(sum(used) + 3)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    starts = _starts(used)
    row = torch.repeat_interleave(torch.arange(len(used), device="cuda"), torch.tensor(used, device="cuda"))
    column = torch.arange(sum(used), device="cuda") - torch.tensor(starts[:-1], device="cuda")[row]
    table[row, column] = order[:sum(used)]
    size = (sum(used) + 3, case["page"], case["kv_heads"], case["dim"])
    dtype = _DTYPE[case["dtype"]]
    return {"lengths": lengths, "kv_lens": _ints(lengths), "table": table, "k_pages": r.normal(*size, dtype=dtype),
            "v_pages": r.normal(*size, dtype=dtype)}


def prepare(case, seed):
    """Inputs ~ N(0, 1) of queries and keys that were normed; buffers for the outputs that a program keeps."""
    r = _Random(seed)
    kind, dtype = case["kind"], _DTYPE[case["dtype"]]
    s = {"case": case}
    if kind == "rotary":
        tokens = case["frames"] * case["rows"] * case["columns"]
        packed = r.normal(tokens, case["heads"] + case["others"], case["dim"], dtype=dtype)
        s["x"] = packed[:, :case["heads"]]  # the queries and keys of a packed projection
        s["positions"] = _grid(0, tokens, case["rows"], case["columns"])
        s["freq"] = _frequencies(case["pairs"])
        s["out"] = torch.empty(s["x"].shape, dtype=dtype, device="cuda")
        return s
    if kind == "norm":
        t, c = case["tokens"], case["channels"]
        s["h"], s["x"] = r.normal(t, c, dtype=dtype, std=2.0), r.normal(t, c, dtype=dtype)
        s["gate"] = r.normal(t // case["gate_tokens"], c, dtype=dtype, std=0.5, mean=0.5)
        s["w_post"], s["w_pre"] = (r.normal(c, dtype=dtype, std=0.2, mean=1.0) for _ in range(2))
        s["x_out"], s["y"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["rstd"] = torch.empty(t, 2, device="cuda")
        if case["step"]:
            s["dx_out"], s["dy"] = r.normal(t, c, dtype=dtype), r.normal(t, c, dtype=dtype)
            s["dh"], s["dx"], s["dgate"] = torch.empty_like(s["x"]), torch.empty_like(s["x"]), torch.empty_like(s["gate"])
            s["dw_post"], s["dw_pre"] = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
        return s
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if kind in ("append", "paged"):
        s.update(_pages(r, case))
        b, new = case["sequences"], case["new"]
        s["cu_q"] = _ints([i * new for i in range(b + 1)])
        packed = r.normal(b * new, hq + 2 * hk, d, dtype=dtype)
        s["q"], s["k"], s["v"] = packed[:, :hq], packed[:, hq:hq + hk], packed[:, hq + hk:]
        if kind == "append":
            s["positions"] = torch.cat([_grid(n - new, new, 45, 80) for n in s["lengths"]])
            s["freq"] = _frequencies(d // 2)
            s["q_out"] = torch.empty(b * new, hq, d, dtype=dtype, device="cuda")
            return s
        s["out"] = torch.empty(b * new, hq, d, dtype=dtype, device="cuda")
        return s
    lengths = _lengths(case)
    s["lengths"], s["cu"] = lengths, _ints(_starts(lengths))
    packed = r.normal(sum(lengths), hq + 2 * hk, d, dtype=dtype)
    s["q"], s["k"], s["v"] = packed[:, :hq], packed[:, hq:hq + hk], packed[:, hq + hk:]
    s["out"] = torch.empty(sum(lengths), hq, d, dtype=dtype, device="cuda")
    s["lse"] = torch.empty(sum(lengths), hq, device="cuda")
    if kind == "train":
        s["dout"] = r.normal(sum(lengths), hq, d, dtype=dtype)
        s["dq"] = torch.empty_like(s["out"])
        s["dk"], s["dv"] = (torch.empty(sum(lengths), hk, d, dtype=dtype, device="cuda") for _ in range(2))
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


def _attention(case):
    return _handle("FrameAttention", case["q_heads"], case["kv_heads"], case["dim"], case["frame"], case["back"], case["ahead"],
                   case["sinks"])


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "rotary":
        op = _handle("Rotary", case["dim"], _sections(case["pairs"]), case["interleaved"])
        op.run_dev(s["x"], s["positions"], s["freq"], s["out"], inverse=case["inverse"])
        return s["out"]
    if kind == "append":
        op = _handle("Rotary", case["dim"], _sections(case["dim"] // 2), False)
        cache = _handle("CacheAppend")
        cache.run_dev(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["cu_q"], s["kv_lens"], rotary=op,
                      positions=s["positions"], freq=s["freq"], q=s["q"], q_out=s["q_out"])
        return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}
    if kind == "norm":
        op = _handle("GatedNorm", case["channels"], case["gate_tokens"], 0.5, _EPS)
        op.forward_dev(s["h"], s["x"], s["gate"], s["w_post"], s["w_pre"], s["x_out"], s["y"], s["rstd"])
        got = {"x_out": s["x_out"], "y": s["y"]}
        if case["step"]:
            op.backward_dev(s["h"], s["x_out"], s["gate"], s["w_post"], s["w_pre"], s["rstd"], s["dx_out"], s["dy"], s["dh"],
                            s["dx"], s["dgate"], s["dw_post"], s["dw_pre"])
            got.update({n: s[n] for n in ("dh", "dx", "dgate", "dw_post", "dw_pre")})
        return got
    op = _attention(case)
    if kind == "paged":
        op.paged_dev(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu_q"], s["kv_lens"], s["out"], max_q=case["new"],
                     max_kv=s["lengths"][0])
        return s["out"]
    longest = s["lengths"][0]
    op.forward_dev(s["q"], s["k"], s["v"], s["out"], s["lse"], cu_q=s["cu"], cu_kv=s["cu"], max_q=longest, max_kv=longest)
    if kind == "attend":
        return {"out": s["out"], "lse": s["lse"]}
    op.backward_dev(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"], s["dv"], cu_q=s["cu"], cu_kv=s["cu"],
                    max_q=longest, max_kv=longest)
    return {n: s[n] for n in ("out", "lse", "dq", "dk", "dv")}


# ---- the plain forms ---------------------------------------------------------------------

def _rotate(x, positions, freq, interleaved, inverse):
    """x [tokens][heads][dim] in 32 bits, turned pair by pair."""
    pairs = freq.numel()
    st, sh, _ = _sections(pairs)
    pair = torch.arange(pairs, device=x.device)
    axis = (pair >= st).long() + (pair >= st + sh).long()
    angle = (positions[:, axis].float() * freq)[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle) * (-1.0 if inverse else 1.0)
    first, second = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + pairs)
    out = x.clone()
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., first] * sin + x[..., second] * cos
    return out


def _visible(n_q, n_kv, max_q, max_kv, case):
    """[sequences][max_q][max_kv]: which key each query sees (n_q, n_kv: the lengths on the GPU)."""
    f = case["frame"]
    i = torch.arange(max_q, device="cuda")[None, :]
    p = (n_kv[:, None] - n_q[:, None] + i)[..., None]
    j = torch.arange(max_kv, device="cuda")[None, None, :]
    seen = (j < n_kv[:, None, None]) & (p >= 0) & (i < n_q[:, None])[..., None]
    fp, fj = torch.div(p, f, rounding_mode="floor"), torch.div(j, f, rounding_mode="floor")
    if case["ahead"] >= 0:
        seen = seen & (fj <= fp + case["ahead"])
    if case["back"] >= 0:
        seen = seen & ((fj >= fp - case["back"]) | (fj < case["sinks"]))
    return seen


def _softmax(scores, seen):
    """The probabilities and the logarithm of the sum, a row that sees nothing having zeros and -inf."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total)), (top + torch.log(total))[..., 0]


def _padded(x, cu, most):
    """[tokens][heads][dim] -> [sequences][heads][most][dim] in 32 bits, zeros past a sequence's end."""
    at = cu[:-1, None].long() + torch.arange(most, device="cuda")
    inside = at < cu[1:, None]
    y = x[torch.where(inside, at, torch.zeros_like(at))].float() * inside[..., None, None]
    return y.transpose(1, 2).contiguous()


def _unpadded(y, cu, tokens):
    """The other way: [sequences][heads][most][dim] -> [tokens][heads][dim]."""
    n = torch.arange(tokens, device="cuda")
    row = torch.searchsorted(cu[1:].contiguous(), n.to(torch.int32), right=True)
    return y.transpose(1, 2)[row, n - cu[row].long()]


def _plain_attention(q, k, v, seen, group):
    """q [B][Hq][mq][D], k and v [B][Hkv][mk][D], all in 32 bits."""
    b, hq, mq, d = q.shape
    hk = hq // group
    grouped = q.reshape(b, hk, group * mq, d)
    scores = torch.matmul(grouped, k.transpose(2, 3)).reshape(b, hk, group, mq, -1) * (1.0 / math.sqrt(d))
    prob, lse = _softmax(scores, seen[:, None, None])
    out = torch.matmul(prob.reshape(b, hk, group * mq, -1), v).reshape(b, hq, mq, d)
    return prob, out, lse.reshape(b, hq, mq)


def _run_plain(s):
    case = s["case"]
    kind, dtype = case["kind"], _DTYPE[case["dtype"]]
    if kind == "rotary":
        return _rotate(s["x"].float(), s["positions"], s["freq"], case["interleaved"], case["inverse"]).to(dtype)
    if kind == "append":
        b, new, page = case["sequences"], case["new"], case["page"]
        k = _rotate(s["k"].float(), s["positions"], s["freq"], False, False).to(dtype)
        q = _rotate(s["q"].float(), s["positions"], s["freq"], False, False).to(dtype)
        at = (s["kv_lens"].long()[:, None] - new + torch.arange(new, device="cuda")).reshape(-1)
        row = torch.arange(b, device="cuda").repeat_interleave(new)
        which = s["table"][row, at // page].long()
        s["k_pages"][which, at % page] = k
        s["v_pages"][which, at % page] = s["v"]
        return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
    if kind == "norm":
        h, x, w1, w2 = (s[n].float() for n in ("h", "x", "w_post", "w_pre"))
        g = s["gate"].float().repeat_interleave(case["gate_tokens"], 0)
        r1 = torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS)
        n1 = h * r1
        xo = x + 0.5 * g * n1 * w1
        r2 = torch.rsqrt((xo * xo).mean(-1, keepdim=True) + _EPS)
        got = {"x_out": xo.to(dtype), "y": (xo * r2 * w2).to(dtype)}
        if case["step"]:
            m, dy = xo * r2, s["dy"].float()
            dm = dy * w2
            t = s["dx_out"].float() + r2 * (dm - m * (dm * m).mean(-1, keepdim=True))
            dn = 0.5 * t * g * w1
            got["dh"] = (r1 * (dn - n1 * (dn * n1).mean(-1, keepdim=True))).to(dtype)
            got["dx"] = t.to(dtype)
            got["dgate"] = (0.5 * t * n1 * w1).reshape(-1, case["gate_tokens"], case["channels"]).sum(1).to(dtype)
            got["dw_post"], got["dw_pre"] = (0.5 * t * g * n1).sum(0), (dy * m).sum(0)
        return got
    group = case["q_heads"] // case["kv_heads"]
    if kind == "paged":
        b, new = case["sequences"], case["new"]
        most = s["table"].shape[1] * case["page"]
        table = s["table"].clamp(min=0).long()
        k, v = (s[n][table].reshape(b, most, case["kv_heads"], case["dim"]).float().transpose(1, 2).contiguous()
                for n in ("k_pages", "v_pages"))
        n_q = s["cu_q"][1:] - s["cu_q"][:-1]
        q = s["q"].reshape(b, new, case["q_heads"], case["dim"]).float().transpose(1, 2).contiguous()
        _, out, _ = _plain_attention(q, k, v, _visible(n_q, s["kv_lens"], new, most, case), group)
        return out.transpose(1, 2).reshape(b * new, case["q_heads"], case["dim"]).to(dtype)
    cu, most, tokens = s["cu"], s["lengths"][0], s["q"].shape[0]
    q, k, v = (_padded(s[n], cu, most) for n in ("q", "k", "v"))
    n = cu[1:] - cu[:-1]
    seen = _visible(n, n, most, most, case)
    prob, out, lse = _plain_attention(q, k, v, seen, group)
    got = {"out": _unpadded(out, cu, tokens).to(dtype), "lse": _unpadded(lse[..., None], cu, tokens)[..., 0]}
    if kind == "attend":
        return got
    b, hq, hk, d = case["sequences"], case["q_heads"], case["kv_heads"], case["dim"]
    do = _padded(s["dout"], cu, most)
    by_kv = lambda x: x.reshape(b, hk, group * most, -1)  # noqa: E731
    prob = by_kv(prob)
    dp = torch.matmul(by_kv(do), v.transpose(2, 3))
    ds = prob * (dp - by_kv((do * out).sum(-1, keepdim=True))) * (1.0 / math.sqrt(d))
    got["dq"] = _unpadded(torch.matmul(ds, k).reshape(b, hq, most, d), cu, tokens).to(dtype)
    got["dk"] = _unpadded(torch.matmul(ds.transpose(2, 3), by_kv(q)), cu, tokens).to(dtype)
    got["dv"] = _unpadded(torch.matmul(prob.transpose(2, 3), by_kv(do)), cu, tokens).to(dtype)
    return got


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- what a pass cannot do without ---------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs, and the keys that any query sees, over the sequences."""
    pairs, keys = 0, 0
    for n in _lengths(case):
        new = case.get("new", n)
        p = np.arange(n - new, n, dtype=np.int64)
        f = p // case["frame"]
        high = np.full_like(p, n) if case["ahead"] < 0 else np.minimum(n, (f + case["ahead"] + 1) * case["frame"])
        low = np.zeros_like(p) if case["back"] < 0 else np.minimum(high, np.maximum(0, (f - case["back"]) * case["frame"]))
        sinks = np.minimum(case["sinks"] * case["frame"], low)
        pairs += int((high - low + sinks).sum())
        keys += int(high.max() - low.min() + np.minimum(sinks.max(), low.min()))
    return pairs, keys


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kind = case["kind"]
    if kind == "rotary":
        tokens = case["frames"] * case["rows"] * case["columns"]
        return {"bytes": tokens * (2 * case["heads"] * case["dim"] * size + 12), "flops": tokens * case["heads"] * case["pairs"] * 6}
    if kind == "norm":
        n = case["tokens"] * case["channels"]
        gates = n // case["gate_tokens"]
        moved = 4 * n + gates + (6 * n + gates if case["step"] else 0)
        return {"bytes": moved * size, "flops": n * (30 if case["step"] else 10)}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        tokens = case["sequences"] * case["new"]
        return {"bytes": tokens * ((2 * hq + 4 * hk) * d * size + 12), "flops": tokens * (hq + hk) * d // 2 * 6}
    pairs, keys = _pairs(case)
    if kind == "paged":
        tokens = case["sequences"] * case["new"]
        return {"bytes": (2 * tokens * hq + 2 * keys * hk) * d * size, "flops": 4 * d * hq * pairs}
    tokens = sum(_lengths(case))
    forward = {"bytes": (2 * tokens * (hq + hk) * d) * size + 4 * tokens * hq, "flops": 4 * d * hq * pairs}
    if kind == "attend":
        return forward
    return {"bytes": forward["bytes"] + (4 * tokens * (hq + hk) * d) * size, "flops": forward["flops"] + 10 * d * hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------

def _exact_turn(x, positions, freq, interleaved, sign):
    st, sh, sw = _sections(freq.numel())
    angle = torch.cat([positions[:, a:a + 1].double() * f for a, f in enumerate(torch.split(freq.double(), [st, sh, sw]))], 1)
    n = freq.numel()
    z = x.double()
    turned, rest = z[..., :2 * n], z[..., 2 * n:]
    pair = turned.unflatten(-1, (n, 2)) if interleaved else turned.unflatten(-1, (2, n)).transpose(-1, -2)
    pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(angle), sign * angle)[:, None])
    pair = pair.flatten(-2) if interleaved else pair.transpose(-1, -2).flatten(-2)
    return torch.cat([pair, rest], -1)


def _exact_mask(n_q, n_kv, case):
    """Sees[i][j] of one sequence, from the intervals of each query's row."""
    place = torch.arange(n_q, device="cuda") + (n_kv - n_q)
    start = place - place % case["frame"]  # the first token of the query's frame
    j = torch.arange(n_kv, device="cuda")[None]
    low = start[:, None] - case["back"] * case["frame"] if case["back"] >= 0 else torch.zeros_like(start[:, None])
    high = start[:, None] + (case["ahead"] + 1) * case["frame"] if case["ahead"] >= 0 else torch.full_like(start[:, None], n_kv)
    return (j < high) & ((j >= low) | (j < case["sinks"] * case["frame"]))


def _exact_head(q, k, v, mask):
    scores = q @ k.T / math.sqrt(q.shape[1])
    scores = scores.masked_fill(~mask, -math.inf)
    return torch.softmax(scores, 1), torch.logsumexp(scores, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_turn(s["x"], s["positions"], s["freq"], case["interleaved"], -1.0 if case["inverse"] else 1.0)
    if kind == "append":
        new, page = case["new"], case["page"]
        k = _exact_turn(s["k"], s["positions"], s["freq"], False, 1.0)
        got = {"q": _exact_turn(s["q"], s["positions"], s["freq"], False, 1.0), "k": s["k_pages"].double(), "v": s["v_pages"].double()}
        for b, n in enumerate(s["lengths"]):
            at = torch.arange(n - new, n, device="cuda")
            slot = s["table"][b].long()[at // page] * page + at % page
            got["k"].flatten(0, 1)[slot] = k[b * new:(b + 1) * new]
            got["v"].flatten(0, 1)[slot] = s["v"][b * new:(b + 1) * new].double()
        return got
    if kind == "norm":
        h, x, gate, w1, w2 = (s[n].double().requires_grad_(case["step"]) for n in ("h", "x", "gate", "w_post", "w_pre"))
        norm = lambda z: z / torch.sqrt(z.square().mean(1, keepdim=True) + _EPS)  # noqa: E731
        by_gate = lambda z: z.reshape(gate.shape[0], -1, case["channels"])  # noqa: E731
        xo = x + (0.5 * gate[:, None] * by_gate(norm(h) * w1)).reshape(x.shape)
        y = norm(xo) * w2
        got = {"x_out": xo.detach(), "y": y.detach()}
        if case["step"]:
            grads = torch.autograd.grad([xo, y], [h, x, gate, w1, w2], [s["dx_out"].double(), s["dy"].double()])
            got.update(zip(("dh", "dx", "dgate", "dw_post", "dw_pre"), grads))
        return got
    group = case["q_heads"] // case["kv_heads"]
    scale = 1.0 / math.sqrt(case["dim"])
    got = {n: torch.empty(s[n].shape, dtype=torch.float64, device="cuda") for n in ("out", "lse", "dq") if n in s}
    got.update({n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("dk", "dv") if n in s})
    starts = _starts(s["lengths"])
    for b, n in enumerate(s["lengths"]):
        new = case.get("new", n)
        rows = slice(b * new, (b + 1) * new) if kind == "paged" else slice(starts[b], starts[b + 1])
        mask = _exact_mask(new, n, case)
        if kind == "paged":
            pages = s["table"][b, :-(-n // case["page"])].long()
            keys, values = (s[p][pages].flatten(0, 1)[:n] for p in ("k_pages", "v_pages"))
        else:
            keys, values = s["k"][rows], s["v"][rows]
        for head in range(case["q_heads"]):
            q, k, v = s["q"][rows, head].double(), keys[:, head // group].double(), values[:, head // group].double()
            prob, lse = _exact_head(q, k, v, mask)
            got["out"][rows, head] = prob @ v
            if "lse" in got:
                got["lse"][rows, head] = lse
            if kind == "train":
                do = s["dout"][rows, head].double()
                slope = prob * (do @ v.T)
                slope = slope - prob * slope.sum(1, keepdim=True)
                got["dq"][rows, head] = slope @ k * scale
                got["dk"][rows, head // group] += slope.T @ q * scale
                got["dv"][rows, head // group] += prob.T @ do
    return got["out"] if kind == "paged" else got
