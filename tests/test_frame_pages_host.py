"""The microscaled cache and shared prefixes without a GPU: the packed structs, what is refused before
the library is called, the workspaces' sizes, and what the copies into LDS rely on."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
import types
from pathlib import Path

import pytest
import torch

from jasnamacos_amd import _lib
from jasnamacos_amd import build as dcn_build
from jasnamacos_amd import frame_attention as fa
from jasnamacos_amd.deform_conv import INVALID_ARGUMENT, INVALID_SHAPE, DeformConvError
from test_frame_attention_device import Library, on, t
from test_frame_attention_host import _copies

BF16, I32, F32, U8 = torch.bfloat16, torch.int32, torch.float32, torch.uint8


def fields(value):
    for name, _ in value._fields_:
        field = getattr(value, name)
        if isinstance(field, C.Structure):
            yield from fields(field)
        elif hasattr(field, "__len__"):
            yield from field
        else:
            yield field


@pytest.mark.parametrize("packed,struct", [(fa._PAGES, _lib.DcnPages), (fa._READ, _lib.DcnReadShape), (fa._PREFIX, _lib.DcnPrefix)])
def test_packed_structs_are_the_c_ones(packed, struct):
    assert packed.size == C.sizeof(struct)
    values = list(range(1, len(packed.unpack(bytes(packed.size))) + 1))
    assert list(fields(struct.from_buffer_copy(packed.pack(*values)))) == values


def _bytes(prefix=None, pages=64, page_tokens=16, width=8, heads=8, dim=64, dtype=1, bits=8, reserved=0, sequences=1, q_heads=8, kv_heads=8,
           head_dim=64, max_q=1, max_kv=128, q_tokens=1):
    lib = _lib.load()
    s = fa._ATTENTION.pack(1, sequences, q_heads, kv_heads, head_dim, 1, -1, 0, 0, max_q, max_kv, 1.0, q_tokens, 0, *[0] * 16)
    p = fa._PAGES.pack(pages, page_tokens, width, heads, dim, dtype, bits, reserved, 0, 0, 0, 0)
    return lib.dcn_attention_pages_workspace_bytes(s, p, prefix and fa._PREFIX.pack(*prefix, 0, 0))


def test_workspace_bytes():
    assert _bytes() == 0  # one part
    long = _bytes(width=4000, max_kv=60000)
    assert long > 0 and long % (8 * (64 + 4) * 4) == 0
    many = dict(sequences=64, q_tokens=64, max_kv=16)
    assert _bytes(**many) == 0
    shared = _bytes((1000, 16000), **many)
    assert shared > 0 and shared % (64 * 8 * (64 + 4) * 4) == 0
    assert _bytes((1000, 0), **many) == 0  # no prefix after all
    assert _bytes((1000, 16000), bits=0, **many) == shared or _bytes((1000, 16000), bits=0, **many) > 0
    other = _bytes(head_dim=96, dim=96, width=4000, max_kv=60000)  # the kernel of any type
    assert other > 0 and other % (8 * (96 + 4) * 4) == 0
    assert _bytes((1000, 16000), head_dim=96, dim=96, max_kv=16) > 0  # parts of the prefix
    assert _bytes(head_dim=96, dim=96, sequences=64, q_tokens=64, width=4000, max_kv=60000) == 0  # workgroups for every CU


@pytest.mark.parametrize("bad", [
    {"bits": 0}, {"bits": 16}, {"bits": 5}, {"reserved": 1}, {"page_tokens": 12}, {"dtype": 0}, {"heads": 4}, {"dim": 128},
    {"head_dim": 40, "dim": 40}, {"prefix": (-1, 0)}, {"prefix": (4, 65)}, {"prefix": (4, -1)}, {"prefix": (1 << 27, 16)},
    {"sequences": -1}, {"max_q": -1}, {"q_heads": 9}])
def test_calls_that_are_refused_need_no_workspace(bad):
    assert _bytes(**{"width": 4000, "max_kv": 60000, **bad}) == 0


def test_keys_that_an_int_counts():
    """Tiles end up to 63 keys past the last one."""
    assert _bytes((2**27 - 4 - 4000, 16), width=4000, max_kv=60000) > 0  # 2^31 - 64 tokens
    assert _bytes((2**27 - 3 - 4000, 16), width=4000, max_kv=60000) == 0


def test_calls_without_a_context_are_refused():
    lib = _lib.load()
    p = fa._PAGES.pack(1, 16, 1, 1, 64, 1, 8, 0, 0, 0, 0, 0)
    s = fa._ATTENTION.pack(1, 1, 1, 1, 64, 1, -1, 0, 0, 1, 1, 1.0, 1, 0, *[0] * 16)
    assert lib.dcn_attention_pages_dev(None, s, p, None, *[None] * 7, 0, None) == INVALID_ARGUMENT
    assert lib.dcn_cache_append_mx_dev(None, p, fa._APPEND.pack(1, 1, 1, *[0] * 8), None, *[None] * 10) == INVALID_ARGUMENT
    assert lib.dcn_cache_read_dev(None, p, fa._READ.pack(1, 0, 1, *[0] * 4), *[None] * 6) == INVALID_ARGUMENT


def u8(*shape):
    return t(*shape, dtype=U8)


def mx(bits=8, dim=64, pages=2, page=16, heads=2):
    return fa.MxPages(u8(pages, heads, page, dim * bits // 8), u8(pages, heads, page, dim * bits // 8), u8(pages, heads, page, dim // 32),
                      u8(pages, heads, page, dim // 32))


def test_buffers():
    for bits in (8, 4):
        p = mx(bits)
        assert (p.bits, p.head_dim, p.kv_heads, p.page_tokens) == (bits, 64, 2, 16)
        z = fa.MxPages.zeros(3, 16, 2, 96, bits, device="cpu")
        assert z.k.shape == (3, 2, 16, 96 * bits // 8) and z.k_scales.shape == (3, 2, 16, 3) and z.bits == bits
    with pytest.raises(AttributeError):
        p.k = u8(1, 1, 1, 1)
    good = [u8(2, 2, 16, 64), u8(2, 2, 16, 64), u8(2, 2, 16, 2), u8(2, 2, 16, 2)]
    fa.MxPages(*good)
    for at, bad, status in ((0, None, INVALID_ARGUMENT), (1, t(2, 2, 16, 64), INVALID_ARGUMENT), (2, u8(2, 2, 16), INVALID_SHAPE),
                            (1, u8(2, 2, 16, 32), INVALID_SHAPE), (3, u8(2, 2, 16, 1), INVALID_SHAPE), (0, u8(2, 2, 16, 48), INVALID_SHAPE),
                            (2, u8(2, 2, 16, 3), INVALID_SHAPE), (1, u8(2, 2, 16, 128)[..., ::2], INVALID_SHAPE),
                            (3, on(1, torch.zeros(2, 2, 16, 2, dtype=U8)), INVALID_ARGUMENT)):
        with pytest.raises(DeformConvError) as e:
            fa.MxPages(*good[:at], bad, *good[at + 1:])
        assert e.value.status == status, (at, e.value.message)
    for sizes in ((1, 16, 1, 48, 8), (1, 16, 1, 0, 8), (1, 16, 1, 64, 16)):
        with pytest.raises(DeformConvError):
            fa.MxPages.zeros(*sizes, device="cpu")


def calls(ctx):
    """name: (call, its arguments)."""
    rotary, attention = fa.Rotary(ctx, 64, (16, 8, 8)), fa.FrameAttention(ctx, 4, 2, 64)
    q, k, lse = t(8, 4, 64), t(8, 2, 64), t(8, 4, dtype=F32)
    table, lens, cu = t(1, 2, dtype=I32), t(1, dtype=I32), t(2, dtype=I32)
    positions, freq, pages = t(8, 3, dtype=I32), t(32, dtype=F32), t(2, 16, 2, 64)
    prefix = {"prefix_table": t(2, dtype=I32), "prefix_len": t(1, dtype=I32)}
    attend = {"q": q, "table": table, "cu_q": cu, "kv_lens": lens, "out": t(8, 4, 64), "lse": lse}
    return {
        "append": (fa.CacheAppend(ctx).run_mx_dev, {"k": k, "v": k, "pages": mx(), "table": table, "cu_q": cu, "kv_lens": lens, "rotary": rotary,
                                                    "positions": positions, "freq": freq, "q": q, "q_out": t(8, 4, 64)}),
        "read": (fa.CacheRead(ctx).run_dev, {"pages": mx(4), "table": table, "cu": cu, "kv_lens": lens, "k_out": k, "v_out": t(8, 2, 64)}),
        "paged": (attention.paged_mx_dev, {"pages": mx(4), **attend}),
        "shared": (attention.shared_dev, {"pages": mx(), **prefix, **attend}),
        "shared as is": (attention.shared_dev, {"pages": (pages, t(2, 16, 2, 64)), **prefix, **attend}),
    }


@pytest.fixture
def ctx():
    lib = Library()
    return types.SimpleNamespace(ctx=None, device=0, _lib=lib, _check=lambda status: None)


NAMES = ["append", "read", "paged", "shared", "shared as is"]


@pytest.mark.parametrize("name", NAMES)
def test_tensors_of_another_device(ctx, name):
    call, args = calls(ctx)[name]
    call(**args)
    assert ctx._lib.calls == 1
    for key, value in args.items():
        if isinstance(value, fa.MxPages):
            others = [fa.MxPages(*(on(where, b.clone()) for b in value._buffers)) for where in (1, -1)]
        elif isinstance(value, tuple):
            others = [(on(1, value[0].clone()), value[1]), (value[0], on(-1, value[1].clone()))]
        elif isinstance(value, torch.Tensor):
            others = [on(where, value.clone()) for where in (1, -1)]
        else:
            continue
        for other in others:
            with pytest.raises(DeformConvError) as e:
                call(**{**args, key: other})
            assert e.value.status == INVALID_ARGUMENT and ctx._lib.calls == 1, key


@pytest.mark.parametrize("name", NAMES)
def test_missing_and_misshapen(ctx, name):
    call, args = calls(ctx)[name]
    optional = {"rotary", "positions", "freq", "lse", "q" if name == "append" else "", "" if name in ("append", "read") else "cu_q"}
    for key, value in args.items():
        bad = [] if key in optional else [None]
        if isinstance(value, torch.Tensor):
            if key not in ("q", "k", "k_out"):
                bad.append(value.to(torch.float64).as_subclass(type(value)))
            if key != "prefix_table":  # of any length
                bad.append(on(0, torch.zeros(tuple(n + 1 for n in value.shape), dtype=value.dtype)))
            bad.append(on(0, torch.zeros((), dtype=value.dtype)))
        for other in bad:
            with pytest.raises(DeformConvError):
                call(**{**args, key: other})
            assert ctx._lib.calls == 0, key
    for key in ("q", "k", "k_out"):  # the type that the others have to be of
        if key in args:
            with pytest.raises(DeformConvError):
                call(**{**args, key: args[key].to(torch.float64).as_subclass(type(args[key]))})
    assert ctx._lib.calls == 0


def test_sizes_outside_their_types(ctx):
    call, args = calls(ctx)["shared"]
    for bound in ({"max_prefix": 2**31}, {"max_q": 2**31}, {"max_kv": -2**31 - 1}):
        with pytest.raises(DeformConvError) as e:
            call(**args, **bound)
        assert e.value.status == INVALID_SHAPE and ctx._lib.calls == 0


@pytest.mark.skipif(shutil.which("hipcc") is None and not Path(dcn_build.HIPCC).exists(), reason="no hipcc")
def test_nothing_else_uses_the_copies_register(tmp_path):
    """The copies set M0 in their own asm without the compiler's knowledge: nothing else may use it."""
    out = tmp_path / "pages.s"
    subprocess.run([dcn_build.HIPCC, "-x", "hip", *dcn_build.DEVICE, *dcn_build.COMMON, "--cuda-device-only", "-S",
                    str(dcn_build.CSRC / "dcn_kernels_attention_pages.hip"), "-o", str(out)], check=True, capture_output=True)
    copies, others = _copies(out.read_text())
    assert copies > 0 and not others


def test_division_by_a_product():
    """The kernels divide 0 .. 2^31 - 1 by sizes as (n * factor) >> shift."""
    for d in [1, 2, 3, 5, 7, 29, 64, 100, 255, 256, 3600, 65535, 65536, 65537, 2**30 - 1, 2**30, 2**30 + 1, 2**31 - 1]:
        bits = (d - 1).bit_length()
        factor, shift = (1 << 31, 31) if d == 1 else ((1 << (31 + bits)) // d + 1, 31 + bits)
        assert factor < 2**32
        for q in {0, 1, 2, (2**31 - 1) // d - 1, (2**31 - 1) // d, 12345 % ((2**31 - 1) // d + 1)}:
            for n in (q * d - 1, q * d, q * d + 1, 2**31 - 1):
                if 0 <= n < 2**31:
                    assert (n * factor) >> shift == n // d, (n, d)
