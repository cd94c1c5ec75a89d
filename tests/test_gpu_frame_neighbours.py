"""No row of FrameAttention's results goes by its neighbours: values that are not finite, or large, reach
the rows that see them and leave the others with the same bits, over the waves of a workgroup, the
tiles of keys and the parts of a sequence."""
from __future__ import annotations

import math

import pytest

import test_gpu_frame_tiles as tiles
from test_gpu_frame_tiles import make, name_of, step, visible

pytestmark = pytest.mark.gpu

CASES = [
    tiles.CASES[0], tiles.CASES[4], tiles.CASES[6], tiles.CASES[9], tiles.PARTS[1][0], tiles.PARTS[2][0], tiles.PARTS[3][0],
    ("bf16", 64, 4, 2, [300, 41], [300, 41], 1, 60, 0, 3),  # 32 rows a workgroup
    ("f16", 128, 4, 2, [200], [200], 1, -1, 0, 0),
    ("f16", 96, 4, 2, [300, 41], [300, 41], 1, 60, 0, 3),  # FP32 products
    ("bf16", 40, 2, 1, [260], [300], 16, 4, 0, 1),
    ("f16", 200, 2, 1, [150], [150], 1, 40, 0, 2),
]


@pytest.mark.parametrize("case", CASES, ids=name_of)
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf, 300.0])
def test_neighbours(case, poison, gpu_ctx):
    """One value of the first sequence. Rows of one workgroup, and of one tile, see it and do not."""
    import torch

    print("case: poison", case, poison, flush=True)
    name, dim, hq, hk, nq, nk, *window = case
    clean = make(case, 4)
    want, _ = step(gpu_ctx, case, clean)
    seen = visible(nq[0], nk[0], *window)
    n, m, at_q, at_k = nq[0], nk[0], nq[0] // 2, nk[0] - nq[0] // 2 - 3
    first = slice(2, 2 + n), slice(2, 2 + m)
    for which, at in (("k", at_k), ("v", at_k), ("q", at_q), ("dout", at_q)):
        d = {key: t.clone() for key, t in clean.items()}
        head = d[which].shape[1] - 1
        d[which][2 + at, head, dim // 3] = poison
        got, _ = step(gpu_ctx, case, d)
        if which in "kv":
            rows, group = seen[:, at], hq // hk
            reached_q = torch.zeros(n, hq, dtype=torch.bool, device="cuda")
            reached_q[rows, head * group:] = True
            keys = seen[rows].any(0)  # that a row sees which the value has reached
        else:
            reached_q = torch.zeros(n, hq, dtype=torch.bool, device="cuda")
            reached_q[at, head] = True
            keys = seen[at]
        reached_k = torch.zeros(m, hk, dtype=torch.bool, device="cuda")
        reached_k[keys, -1] = True
        for key in ("out", "lse", "dq"):
            assert torch.equal(got[key][first[0]][~reached_q], want[key][first[0]][~reached_q]), (which, key)
        for key in ("dk", "dv"):
            assert torch.equal(got[key][first[1]][~reached_k], want[key][first[1]][~reached_k]), (which, key)
        for key in want:  # the other sequences
            rest = slice(2 + n, -1) if key in ("out", "lse", "dq") else slice(2 + m, -1)
            assert torch.equal(got[key][rest], want[key][rest]), (which, key)
        finite = {key: torch.isfinite(got[key].float()) for key in got}
        if (which == "v" and not math.isfinite(poison)) or (which == "k" and math.isnan(poison)):  # (a score of -inf is a weight of 0)
            assert reached_q.any() and not finite["out"][first[0]][reached_q].all(1).any(), which
            assert not finite["dq"][first[0]][reached_q].all(1).any()
        if which == "dout" and not math.isfinite(poison):
            assert not finite["dv"][first[1]][reached_k].all(1).any()
