"""Attention over a prefix that is read once for all sequences, in pages of the type and in codes of 8 and 4 bits:
blocks of 16, 32 and 128 rows over the prefix and over the sequences' own keys, against the definition in
64 bits. That the cases are shared out so is tested without a GPU (test_frame_pages_rules.py)."""
from __future__ import annotations

import pytest
import torch

from frame_pages_cases import BITS, READ_ONCE, Call, name_of, scaled

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    from jasnamacos_amd import frame_attention

    return frame_attention


@pytest.mark.parametrize("which", range(len(READ_ONCE)), ids=lambda i: f"{READ_ONCE[i][0]}-{name_of(READ_ONCE[i][1])}")
@pytest.mark.parametrize("bits", BITS)
def test_read_once(fa, gpu_ctx, which, bits):
    case = scaled(READ_ONCE[which][1], bits)
    print("case: read once", READ_ONCE[which][0], name_of(case), bits, flush=True)
    call = Call(case, bits)
    out, lse = call.run(fa, gpu_ctx)
    call.compare(out, lse)
    again = call.run(fa, gpu_ctx)
    assert torch.equal(again[0].nan_to_num(7.0), out.nan_to_num(7.0)) and torch.equal(again[1].nan_to_num(7.0), lse.nan_to_num(7.0))


@pytest.mark.parametrize("which", [1, 2, 4, 5, 7, 9, 10], ids=lambda i: f"{READ_ONCE[i][0]}-{name_of(READ_ONCE[i][1])}")
@pytest.mark.parametrize("bits", BITS)
def test_unseen_and_missing(fa, gpu_ctx, which, bits):
    """A page of the prefix and one of a sequence that are not there; NaN where only some of the rows look, in the
    prefix and in a sequence's own keys."""
    case = scaled(READ_ONCE[which][1], bits)
    print("case: read once, unseen", READ_ONCE[which][0], name_of(case), bits, flush=True)
    page, prefix, nq, nk = case[4:8]
    call = Call(case, bits)
    tables = {"prefix_table": call.prefix_table.clone(), "table": call.table.clone()}
    s = max(call.sequences(), key=lambda t: nk[t])
    tables["prefix_table"][3], tables["table"][s, 0] = -1, 1 << 30
    out, lse = call.run(fa, gpu_ctx, **tables)
    call.compare(out, lse, gone={-1: [3], s: [0]})
    counts = sum(call.seen(t)[:, :prefix].sum(0) for t in range(len(nq)))
    some = ((counts > 0) & (counts < sum(nq))).nonzero().flatten()
    some = some[(some // page) != 3]
    for j in {int(some[len(some) // 2]) if len(some) else prefix - 1, 0}:
        call.unseen(fa, gpu_ctx, out, lse, 0, j, **tables)
    t = min(call.sequences(), key=lambda t: (t == s, -nk[t]))
    if nk[t]:
        call.unseen(fa, gpu_ctx, out, lse, t, prefix + nk[t] - 1, **tables)
