"""What the kernels of attention over pages compute of positions, on the host: the library's own functions,
compiled into a small program."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from jasnamacos_amd import build as dcn_build

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
