"""Frame attention without a GPU: the packed structs, the workspaces' sizes, and what the
copies into LDS rely on in the generated code."""
from __future__ import annotations

import concurrent.futures
import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from jasnamacos_amd import _lib
from jasnamacos_amd import build as dcn_build
from jasnamacos_amd import frame_attention as fa


@pytest.mark.parametrize("packed,struct", [
    (fa._ROTARY, _lib.DcnRotary), (fa._CACHE, _lib.DcnCache), (fa._APPEND, _lib.DcnAppendShape),
    (fa._ATTENTION, _lib.DcnAttentionShape), (fa._NORM, _lib.DcnNormShape)])
def test_packed_structs_are_the_c_ones(packed, struct):
    """Distinct values packed in order come back from the fields in order."""
    assert packed.size == C.sizeof(struct)
    values = list(range(1, len(packed.unpack(bytes(packed.size))) + 1))
    got = struct.from_buffer_copy(packed.pack(*values))
    flat = []
    for name, _ in struct._fields_:
        field = getattr(got, name)
        flat += list(field) if hasattr(field, "__len__") else [field]
    assert flat == values


def _bytes(which, dtype=1, sequences=1, q_heads=8, kv_heads=8, dim=64, max_q=1, max_kv=1, q_tokens=1, kv_tokens=1):
    lib = _lib.load()
    s = fa._ATTENTION.pack(dtype, sequences, q_heads, kv_heads, dim, 1, -1, 0, 0, max_q, max_kv, 1.0, q_tokens, kv_tokens,
                           *[0] * 16)
    return lib.dcn_attention_workspace_bytes(s, which)


def test_workspace_bytes():
    assert _bytes(fa.PASS_FORWARD, dtype=2) == 0  # FP32 heads need none
    assert _bytes(fa.PASS_FORWARD, max_kv=64, kv_tokens=64) == 0  # one part
    split = _bytes(fa.PASS_FORWARD, max_kv=100000, kv_tokens=100000)
    assert split > 0 and split % (8 * (64 + 4) * 4) == 0
    # The backward keeps a delta of four bytes for each row and head.
    assert _bytes(fa.PASS_BACKWARD, dtype=2, q_tokens=33, max_q=33) == 33 * 8 * 4
    assert _bytes(fa.PASS_BACKWARD, q_tokens=33, max_q=33) >= 33 * 8 * 4


@pytest.mark.parametrize("bad", [
    {"dtype": 3}, {"dtype": -1}, {"sequences": -1}, {"sequences": 65536}, {"q_heads": 3, "kv_heads": 2}, {"dim": 0},
    {"dim": 257}, {"max_q": -1}, {"q_tokens": -1}, {"max_q": 2**31 - 1, "q_tokens": 2**31}])
def test_shapes_that_are_refused_need_no_workspace(bad):
    assert _bytes(fa.PASS_BACKWARD, **bad) == 0


def test_calls_without_a_context_are_refused():
    lib = _lib.load()
    s = fa._ATTENTION.pack(1, 1, 1, 1, 64, 1, -1, 0, 0, 1, 1, 1.0, 1, 1, *[0] * 16)
    none = [None] * 7
    assert lib.dcn_attention_forward_dev(None, s, *none, None, 0, None) == 7


def _copies(asm: str) -> tuple[int, list[str]]:
    """(copies into LDS, uses of M0 that are not such a copy's)."""
    lines = [t for t in (x.split(";")[0].strip() for x in asm.splitlines()) if t and not t.startswith((".", "#"))]
    copies, others = 0, []
    for i, t in enumerate(lines):
        if t.startswith("global_load_lds"):
            copies += 1
            if not (lines[i - 2].startswith("s_mov_b32 m0,") and lines[i - 1] == "s_nop 0"):
                others.append(t)
        elif re.search(r"\bm0\b", t) and not (t.startswith("s_mov_b32 m0,") and lines[i + 2].startswith("global_load_lds")):
            others.append(t)
    return copies, others


def test_copy_detector():
    good = "s_mov_b32 m0, s4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 v1, s[2:3]\n"
    assert _copies(good) == (1, [])
    assert _copies(good + "s_mov_b32 m0, 0\nv_readlane_b32 s1, v2, m0\ns_endpgm\n")[1]
    assert _copies("s_nop 0\ns_nop 0\nglobal_load_lds_dwordx4 v1, s[2:3]\n")[1]


@pytest.mark.skipif(shutil.which("hipcc") is None and not Path(dcn_build.HIPCC).exists(), reason="no hipcc")
def test_nothing_else_uses_the_copies_register(tmp_path):
    """The copies set M0 in their own asm without the compiler's knowledge: nothing else may use it."""
    def asm(name):
        out = tmp_path / f"{name}.s"
        subprocess.run([dcn_build.HIPCC, "-x", "hip", *dcn_build.DEVICE, *dcn_build.COMMON, "--cuda-device-only", "-S",
                        str(dcn_build.CSRC / name), "-o", str(out)], check=True, capture_output=True)
        return _copies(out.read_text())
    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        for copies, others in pool.map(asm, ["dcn_kernels_attention.hip", "dcn_kernels_attention_backward.hip"]):
            assert copies > 0 and not others
