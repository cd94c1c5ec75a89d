"""64-bit definitions of the frame-attention operators, on the CPU, and bounds on how far a
result in fewer bits may be from them.

Bounds are worst cases, summed from each rounding: u is half the distance between 1 and the
next number of a type (a rounding's relative error), an FP32 dot product of n terms is off
by at most n 2^-24 of the sum of its terms' magnitudes."""
from __future__ import annotations

import math

import torch

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
# Half of a type's smallest step: what the rounding of a subnormal result may be off by.
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}


def visible(nq, nk, frame, back, ahead, sinks):
    """[nq][nk] truth values, straight from the definition."""
    seen = torch.zeros(nq, nk, dtype=torch.bool)
    for i in range(nq):
        p = nk - nq + i
        if p < 0:
            continue
        f = p // frame
        for j in range(nk):
            fj = j // frame
            seen[i, j] = (ahead < 0 or fj <= f + ahead) and (back < 0 or fj >= f - back or fj < sinks)
    return seen


def attention(q, k, v, seen, scale, dtype, dout=None):
    """One head: values in 64 bits and, for each output, the bound on a `dtype` result."""
    q, k, v = (t.double() for t in (q, k, v))
    u, tiny, dim, nk = U[dtype], TINY[dtype], q.shape[1], k.shape[0]
    s = (q @ k.T) * scale
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))[:, None]) * seen
    out = p @ v
    # Scores: a dot product's error, the scale folded in and two roundings, magnified by exp.
    # P: that error twice (score and sum), the sum's own, and one rounding to 16 bits.
    size = (q.abs() @ k.abs().T).max().item() * abs(scale) if nk and len(q) else 0.0
    ds = (dim + 6) * 2.0**-24 * size
    e = 4 * ds + (nk + 16) * 2.0**-23
    got = {"out": (out, (2 * u + e) * (p @ v.abs()) + tiny), "lse": (lse, torch.full_like(lse, ds + 2.0**-20) + 2.0**-20 * lse.abs().nan_to_num(0, 0, 0))}
    if dout is None:
        return got
    do = dout.double()
    dp = do @ v.T
    delta = (do * out).sum(1, keepdim=True)
    t = p * (dp - delta)
    # dS: its factors' errors (delta is taken from the rounded out) and its own rounding.
    err = (u + e) * t.abs() + p * ((dim + 4) * 2.0**-23 * (do.abs() @ v.abs().T) + (u + e + dim * 2.0**-23)
                                   * (do.abs() * (p @ v.abs())).sum(1, keepdim=True))
    n = nk + len(q)
    grow = 1 + 2 * n * 2.0**-24
    got["dq"] = (t @ k * scale, abs(scale) * (err @ k.abs()) * grow + (u + n * 2.0**-23) * abs(scale) * (t.abs() @ k.abs()) + tiny)
    got["dk"] = (t.T @ q * scale, abs(scale) * (err.T @ q.abs()) * grow + (u + n * 2.0**-23) * abs(scale) * (t.abs().T @ q.abs()) + tiny)
    got["dv"] = (p.T @ do, (2 * u + e + n * 2.0**-23) * (p.T @ do.abs()) + tiny)
    return got


def rotate(x, positions, freq, pairs, interleaved, inverse):
    """[tokens][heads][dim] in 64 bits."""
    n = sum(pairs)
    axis = [0] * pairs[0] + [1] * pairs[1] + [2] * pairs[2]
    angle = positions.double()[:, axis] * freq.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None] * (-1 if inverse else 1)
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + (1 if interleaved else n)
    out = x.double().clone()
    a, b = x.double()[..., first], x.double()[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    return out


def gated_norm(h, x, gate, w_post, w_pre, gate_tokens, scale, eps):
    """(x_out, y) in 64 bits; None gates and weights are ones."""
    norm = lambda z: z / torch.sqrt((z * z).mean(1, keepdim=True) + eps)  # noqa: E731
    u = norm(h)
    if w_post is not None:
        u = u * w_post
    if gate is not None:
        u = u * gate.repeat_interleave(gate_tokens, 0)[: len(h)]
    x_out = x + scale * u
    y = norm(x_out)
    return x_out, y if w_pre is None else y * w_pre
