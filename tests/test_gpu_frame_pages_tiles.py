"""Blocks of 128 rows over a sequence's own pages (of the type, and in codes of 8 and 4 bits), and over a prefix
before them that each block reads for itself, against the definition in 64 bits. That the cases take such
blocks is tested without a GPU (test_frame_pages_rules.py)."""
from __future__ import annotations

import pytest
import torch

from frame_pages_cases import BITS, TILES, Call, name_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


@pytest.mark.parametrize("case", TILES, ids=name_of)
@pytest.mark.parametrize("bits", BITS)
def test_tiles(fa, gpu_ctx, case, bits):
    print("case: tiles", name_of(case), bits, flush=True)
    call = Call(case, bits)
    out, lse = call.run(fa, gpu_ctx)
    call.compare(out, lse)
    again = call.run(fa, gpu_ctx)
    assert torch.equal(again[0].nan_to_num(7.0), out.nan_to_num(7.0)) and torch.equal(again[1].nan_to_num(7.0), lse.nan_to_num(7.0))


@pytest.mark.parametrize("case", TILES, ids=name_of)
@pytest.mark.parametrize("bits", BITS)
def test_unseen_and_missing(fa, gpu_ctx, case, bits):
    """Pages that are not there, and NaN in keys and values that only some rows of a block see."""
    print("case: tiles, unseen", name_of(case), bits, flush=True)
    page, prefix, nq, nk = case[4:8]
    call = Call(case, bits)
    s = max(call.sequences(), key=lambda t: nk[t])
    tables, gone = {"table": call.table.clone()}, {s: [1, (nk[s] - 1) // page]}
    tables["table"][s, 1], tables["table"][s, gone[s][1]] = -(1 << 31), call.buffers[0].shape[0]
    if prefix:
        tables["prefix_table"] = call.prefix_table.clone()
        tables["prefix_table"][1], gone[-1] = 1 << 30, [1]
    out, lse = call.run(fa, gpu_ctx, **tables)
    call.compare(out, lse, gone)
    missing = lambda t, j: (j // page in gone.get(-1, ())) if j < prefix else ((j - prefix) // page in gone.get(t, ()))  # noqa: E731
    for t in {s, min(call.sequences(), key=lambda t: (t == s, -nq[t]))}:
        seen = call.seen(t)
        some = [j for j in (seen.any(0) & ~seen.all(0)).nonzero().flatten().tolist() if not missing(t, j)]
        if not some:  # every row sees every key, or none
            some = [j for j in range(prefix + nk[t]) if not missing(t, j)]
        for j in {some[len(some) // 2], some[-1]} if some else ():
            call.unseen(fa, gpu_ctx, out, lse, t, j, **tables)
