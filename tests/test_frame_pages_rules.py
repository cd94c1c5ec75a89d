"""What the kernels of attention over pages compute of positions, and how a call is shared out among them, on the
host: the library's own functions, compiled into a small program."""
from __future__ import annotations

import random
import shutil
import subprocess
from pathlib import Path

import pytest

from jasnamacos_amd import _lib
from jasnamacos_amd import build as dcn_build
from jasnamacos_amd import frame_attention as fa
from frame_pages_cases import BITS, READ_ONCE, TILES, name_of, rows_of, scaled

LAST = 2**31 - 1
SOURCE = Path(__file__).resolve().parent / "cpp" / "attention_pages_host.hip"

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not Path(dcn_build.HIPCC).exists(), reason="no hipcc")


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    """ask(lines): the program's answers, a list of whole numbers each."""
    program = tmp_path_factory.mktemp("pages") / "attention_pages_host"
    subprocess.run([dcn_build.HIPCC, "-x", "hip", "--cuda-host-only", *dcn_build.DEVICE, *dcn_build.COMMON, "-O1", str(SOURCE), "-o", str(program)],
                   check=True, capture_output=True)

    def run(lines):
        lines = list(lines)
        out = subprocess.run([str(program)], input="\n".join(lines), text=True, capture_output=True, check=True).stdout.splitlines()
        assert len(out) == len(lines)
        return [[int(v) for v in line.split()] for line in out]
    return run


def span(frame, ahead, back, sinks, p, n):
    """The definition, in whole numbers of any size: keys [0, sink) and [lo, hi)."""
    if p < 0:
        return [0, 0, 0]
    f = p // frame
    hi = n if ahead < 0 else min(n, (f + ahead + 1) * frame)
    lo = 0 if back < 0 else min(hi, max(0, (f - back) * frame))
    return [min(sinks * frame, lo), lo, hi]


def test_windows_next_to_the_largest_numbers(ask):
    """Windows whose ends lie at, before and past 2^31 - 1 tokens: what a position sees is what the definition
    says, in the kernels of any type and in the others."""
    cases = []
    for frame in (1, 2, 3, 64, 3600, 2**15, 2**16 + 1, 2**29, 2**30 - 1, 2**30, 2**30 + 1, LAST - 64, LAST):
        most = LAST // frame
        counts = {c for c in (0, 1, most // 2, most - 2, most - 1, most, most + 1, LAST) if 0 <= c <= LAST}
        places = {p for p in (-1, 0, 1, frame - 1, frame, frame + 1, most * frame - frame - 1, most * frame - frame, most * frame - 1, most * frame,
                              LAST - 65, LAST - 1) if -1 <= p < LAST}
        lengths = {n for n in (0, 1, frame, frame + 5, most * frame - 1, most * frame, most * frame + 5, LAST - 64, LAST) if 0 <= n <= LAST}
        for count in counts:
            for p in places:
                for n in lengths:
                    cases += [(frame, count, -1, 0, p, n), (frame, -1, count, 1, p, n), (frame, 0, 0, count, p, n), (frame, count, 1, count, p, n)]
    for case, got in zip(cases, ask("window " + " ".join(map(str, c)) for c in cases)):
        want = span(*case)
        assert got[3:] == want, ("any type", case, got, want)
        assert got[:3] == want, (case, got, want)


def test_division_by_sizes(ask):
    """0 .. 2^31 - 1 by any number from 1 on, at multiples, next to them and at random."""
    r = random.Random(1)
    sizes = {1, 2, 3, 5, 6, 7, 29, 64, 100, 255, 256, 3600, 65535, 65536, 65537, 2**30 - 1, 2**30, 2**30 + 1, LAST - 1, LAST}
    sizes |= {r.randint(1, 2**r.randint(1, 31) - 1) for _ in range(200)}
    pairs = []
    for d in sorted(sizes):
        for q in {0, 1, 2, LAST // d - 1, LAST // d, r.randint(0, LAST // d), r.randint(0, LAST // d)}:
            pairs += [(d, n) for n in (q * d - 1, q * d, q * d + 1, r.randint(0, LAST), LAST) if 0 <= n <= LAST]
    for (d, n), got in zip(pairs, ask(f"divide {d} {n}" for d, n in pairs)):
        assert got == [n // d], (n, d)


class Plan:
    def __init__(self, values):
        self.shared, self.both, self.parts, self.rows, self.waves, self.blocks, self.splits = values[:7]
        self.prefix_rows, self.prefix_waves, self.prefix_blocks, self.prefix_splits, self.prefix_grid, self.grid, self.fits = values[7:]


def plan(ask, dim, bits, hq, hk, nq, nk, prefix, frame, back, sinks, q_tokens):
    """How a call with these lengths as its bounds is shared out."""
    max_q = min(max(nq), q_tokens)
    return Plan(ask([f"plan {dim} {bits} {len(nq)} {hk} {hq // hk} {q_tokens} {max_q} {max(nk)} {prefix} {frame} {back} {sinks}"])[0])


@pytest.mark.parametrize("bits", [0, 8, 4])
@pytest.mark.parametrize("sequences,keys,prefix", [(64, 16, 16000), (64, 16, 60000), (1, 60000, 0), (1, 60000, 900), (300, 200, 500)])
def test_workspaces_have_room_for_the_parts(ask, bits, sequences, keys, prefix):
    """FP32 of each part of a row: its channels, a maximum and a sum, in a line of four more."""
    lib = _lib.load()
    s = fa._ATTENTION.pack(1, sequences, 8, 8, 64, 1, -1, 0, 0, 1, keys, 1.0, sequences, 0, *[0] * 16)
    p = fa._PAGES.pack(64, 16, 4000, 8, 64, 1, bits, 0, 0, 0, 0, 0)
    size = lib.dcn_attention_pages_workspace_bytes(s, p, fa._PREFIX.pack(4000, prefix, 0, 0))
    got = plan(ask, 64, bits, 8, 8, [1] * sequences, [keys], prefix, 1, -1, 0, sequences)
    assert size == (0 if got.parts == 1 else sequences * 8 * got.parts * (64 + 4) * 4)
    assert got.shared == ((sequences - 1) * prefix * 8 * 64 * (bits or 16) / 4 > 120e6)
    assert got.parts == got.splits + got.shared * got.prefix_splits and (got.parts > 1 or not got.shared)


def plan_of(ask, case, bits):
    name, dim, hq, hk, page, prefix, nq, nk, frame, back, ahead, sinks = case
    return plan(ask, dim, bits, hq, hk, nq, nk, prefix, frame, back, sinks, rows_of(case))


@pytest.mark.parametrize("bits", BITS)
def test_cases_that_are_read_once(ask, bits):
    for (prefix_rows, rows), case in READ_ONCE:
        got = plan_of(ask, scaled(case, bits), bits)
        assert (got.shared, got.prefix_rows, got.rows) == (1, prefix_rows, rows), (name_of(case), vars(got))


@pytest.mark.parametrize("bits", BITS)
def test_cases_of_128_rows(ask, bits):
    for case in TILES:
        got = plan_of(ask, case, bits)
        assert (got.shared, got.both, got.rows) == (0, case[5] > 0, 128), (name_of(case), vars(got))


def test_launches_of_less_than_2_24_workgroups(ask):
    """They fit, whatever the threads of a workgroup, as every launch has fewer than 2^32 threads; larger ones do not."""
    for dim in (64, 128):
        for bits in BITS:
            for sequences, heads, new in ((65535, 65, 1), (65535, 255, 1), (65535, 250, 17), (60000, 2, 16000), (1, 3, 600_000_000)):
                got = plan(ask, dim, bits, heads, heads, [new] * sequences, [50], 0, 1, -1, 0, sequences * new)
                assert got.grid < 2**24 and got.grid * 64 * got.waves < 2**32 and got.fits, (dim, bits, sequences, heads, new, vars(got))
            for sequences, heads, new in ((65535, 258, 1), (65535, 65535, 1), (65535, 100, 3000)):
                assert not plan(ask, dim, bits, heads, heads, [new] * sequences, [50], 0, 1, -1, 0, sequences * new).fits
            # A prefix that is read once, and the join of its parts.
            for sequences, heads, fits in ((60, 65535, 1), (16000, 500, 1), (65535, 65535, 0)):
                got = plan(ask, dim, bits, heads, heads, [1] * sequences, [50], 4000, 1, -1, 0, sequences)
                assert got.shared and got.fits == fits, (dim, bits, sequences, heads, vars(got))
            for heads, queries, fits in ((50000, 120, 1), (65535, 127, 1)):  # rows to join: up to 2^23
                got = plan(ask, dim, bits, heads, heads, [queries] * 2, [50], 100, 1, -1, 0, 2 * queries)
                assert got.shared and got.fits == fits and got.parts > 1, (dim, bits, heads, vars(got))


@pytest.mark.parametrize("pages,page_tokens,heads", [(LAST, 2**30, 8), (LAST, 64, 8), (2**20, 512, 8), (LAST // (8 * 16) + 1, 16, 8)])
def test_pools_of_more_rows_than_an_int_counts(pages, page_tokens, heads):
    """They take the kernel of any type, whose rows have 64 bits: the workspace is for its parts. (2^31 - 1 pages
    of 2^30 tokens of 8 heads are more than 64 bits count.)"""
    def size(**sizes):
        s = fa._ATTENTION.pack(1, 1, heads, heads, sizes.get("dim", 64), 1, -1, 0, 0, 1, 2000, 1.0, 1, 0, *[0] * 16)
        p = fa._PAGES.pack(sizes.get("pages", pages), sizes.get("page_tokens", page_tokens), 2**20 if page_tokens < 1024 else 1, heads,
                           sizes.get("dim", 64), 1, 8, 0, 0, 0, 0, 0)
        return _lib.load().dcn_attention_pages_workspace_bytes(s, p, None)
    line = lambda dim: (dim + 4) * 4 * heads  # noqa: E731
    assert size(pages=4, page_tokens=64) == 0  # the matrix kernels: one workgroup a head
    assert size() == size(dim=96) // line(96) * line(64) > 0


def test_rows_that_lie_on_others(ask):
    """Against the places themselves, for tensors that lie in memory in many ways."""
    r = random.Random(2)
    questions, want = [], []
    for _ in range(4000):
        tokens, dim, size = r.randint(1, 6), r.choice([1, 2, 4]), r.choice([2, 4])
        in_heads, out_heads = r.randint(1, 5), r.randint(1, 5)
        hs = dim + r.choice([0, 0, 1, 5])
        ts = r.choice([1, 2, 3]) * (max(in_heads, out_heads) * hs + r.choice([0, 1]))
        if r.random() < 0.3:  # heads first
            hs, ts = tokens * dim + r.choice([0, 2]), dim
        in_s = (0 if r.random() < 0.1 else ts, 0 if r.random() < 0.1 else hs)
        apart = r.randint(-3 * ts * tokens, 3 * ts * tokens) if r.random() < 0.5 else r.choice([-1, 1]) * r.choice([0, hs, in_heads * hs, out_heads * hs])
        places = lambda at, s, heads: {at + i * s[0] + h * s[1] + c for i in range(tokens) for h in range(heads) for c in range(dim)}  # noqa: E731
        meets = bool(places(0, in_s, in_heads) & places(apart, (ts, hs), out_heads))
        same = (tokens == 1 or in_s[0] == ts) and (in_heads == out_heads == 1 or in_s[1] == hs)
        if not same and not meets:
            continue  # other strides: rows in between may count as met
        questions.append(f"meet {1 << 20} {in_s[0]} {in_s[1]} {in_heads} {(1 << 20) + apart * size} {ts} {hs} {out_heads} {tokens} {dim} {size}")
        want.append([int(meets)])
    assert 500 < sum(w[0] for w in want) < len(want) - 500
    for question, w, got in zip(questions, want, ask(questions)):
        assert got == w, question
    # Sizes that a product of 64 bits does not hold, and tensors apart of other strides.
    big, far = 2**40 - 1, 1 << 46
    assert ask([f"meet 64 {big} 64 1 {64 + 2**33} {big} 64 1 {LAST} 64 2", f"meet 64 {big} 64 1 {64 + 2 * big * 1000} {big} 64 1 {LAST} 64 2",
                f"meet 64 1536 64 8 {far} 512 64 8 100000 64 2", f"meet {far} 512 64 8 64 1536 64 8 100000 64 2",
                f"meet 64 1536 64 8 {64 + 2 * 1024} 512 64 8 100000 64 2"]) == [[0], [1], [0], [0], [1]]
