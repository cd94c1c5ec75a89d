"""Frame attention over libdcn: the operators of a block in which the tokens of a clip's
frames attend to the frames before them.

  Rotary          rotary positions with three axes (time, height, width), and their gradient
  CacheAppend     new keys and values into a paged cache, rotated on the way
  MxPages         the buffers of a microscaled cache: codes of 8 or 4 bits, a power of two for 32
  CacheRead       a microscaled cache read back
  FrameAttention  attention over a window of frames with the first ones kept visible:
                  forward, backward, over the paged cache, and for streams that share a prefix
  GatedNorm       the norms after and before a block, its gate and its residual scale

No counterpart in the reference. Tensors are torch tensors on the context's device;
tensors of heads are [tokens][heads][channels] with adjacent channels, so a slice of a
packed projection is taken as it is. As elsewhere in this package outputs are the caller's,
calls are asynchronous on `stream` (None: the default stream), and errors are
DeformConvError. A FrameAttention or GatedNorm keeps the workspace of its calls: calls that
may run at the same time need a handle each, and a handle sizes its workspace in its first
call of a size (reserve it before a graph capture by running that call once). A workspace that
a larger call has replaced stays with the handle, since a captured graph may still use it. Keep
a handle as long as the graphs captured with it, and until its calls on streams other than
torch's current one have ended."""
from __future__ import annotations

import ctypes as C
import math
import struct

import torch

from . import _lib
from .deform_conv import INVALID_ARGUMENT, INVALID_SHAPE, DeformConvError, HipDeformConv, _ptr, _stream

DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
PASS_FORWARD, PASS_BACKWARD, PASS_PAGED = 0, 1, 2


def _dtype(t) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise DeformConvError(INVALID_ARGUMENT, f"dtype {t.dtype} is not float16, bfloat16 or float32")
    return code


def _need(condition, message: str) -> None:
    if not condition:
        raise DeformConvError(INVALID_SHAPE, message)


def _on_device(name: str, t, device: int) -> None:
    if t is None:
        raise DeformConvError(INVALID_ARGUMENT, f"{name} is missing")
    if not t.is_cuda:
        raise DeformConvError(INVALID_ARGUMENT, f"{name} is not on a device")
    if t.get_device() != device:
        raise DeformConvError(INVALID_ARGUMENT, f"{name} is on device {t.get_device()}; the context is on {device}")


def _heads(name: str, t, dtype, shape, device: int) -> tuple:
    """The strides of a tensor of heads of this shape."""
    if t is not None and t.shape == shape and t.dtype is dtype and t.get_device() == device:
        strides = t.stride()
        if strides[2] == 1 or shape[2] == 1:
            return strides
        raise DeformConvError(INVALID_SHAPE, f"{name} channels are not adjacent")
    _on_device(name, t, device)
    if t.dtype is not dtype:
        raise DeformConvError(INVALID_ARGUMENT, f"{name} is {t.dtype}; expected {dtype}")
    raise DeformConvError(INVALID_SHAPE, f"{name} is {tuple(t.shape)}; expected {shape}")


def _rows(name: str, t) -> int:
    """The rows of a tensor of heads."""
    if t is None:
        raise DeformConvError(INVALID_ARGUMENT, f"{name} is missing")
    if t.dim() != 3:
        raise DeformConvError(INVALID_SHAPE, f"{name} has {t.dim()} dimensions; expected [tokens][heads][channels]")
    return t.shape[0]


def _whole(name: str, t, dtype, shape, device: int) -> None:
    """An adjacent tensor of this type and shape."""
    if t is not None and t.shape == shape and t.dtype is dtype and t.is_contiguous() and t.get_device() == device:
        return
    _on_device(name, t, device)
    if t.dtype is not dtype:
        raise DeformConvError(INVALID_ARGUMENT, f"{name} is {t.dtype}; expected {dtype}")
    raise DeformConvError(INVALID_SHAPE, f"{name} is {tuple(t.shape)}; expected {shape}, adjacent")


def _index(name: str, t, count, device: int) -> None:
    """An adjacent int32 array of this length."""
    if t is not None and t.dtype is torch.int32 and t.shape == (count,) and t.is_contiguous() and t.get_device() == device:
        return
    _on_device(name, t, device)
    raise DeformConvError(INVALID_SHAPE, f"{name} is not {count} adjacent int32 values")


# The C structs' layouts: packing one is several times faster than filling its fields.
_ROTARY = struct.Struct("6i")
_CACHE = struct.Struct("6i")
_APPEND = struct.Struct("iiq8q")
_ATTENTION = struct.Struct("11ifqq16q")
_PAGES = struct.Struct("8i4Q")
_AS_IS = struct.Struct("2i4Q")  # of a dcn_pages, what follows its dcn_cache
_READ = struct.Struct("iiq4q")
_PREFIX = struct.Struct("2i2Q")
_NORM = struct.Struct("iiqqff")
_NO_STRIDES = (0, 0)


def _outside() -> DeformConvError:
    """For a size that its C type does not hold (struct.error of a layout above)."""
    return DeformConvError(INVALID_SHAPE, "a size is outside its C type")


def _factor(name: str, value) -> float:
    """A number that FP32 holds (packing one that it does not gives an infinity)."""
    value = float(value)
    _need(abs(value) <= torch.finfo(torch.float32).max, f"{name} is not a finite FP32 number")
    return value


def _fresh(count: int, like):
    """Memory for a handle. The allocator may hand out what work on the current stream still
    reads; the handle's calls may be on another one."""
    t = torch.empty(count, dtype=torch.uint8, device=like.device)
    if not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(like.device).synchronize()
    return t


class _Handle:
    def __init__(self, ctx: HipDeformConv):
        self.ctx = ctx
        self._ctx = ctx.ctx
        self._lib = ctx._lib
        self._workspace = None
        self._replaced = []  # memory that larger calls have outgrown: graphs may hold its address
        self._sizes = {}  # workspace bytes of the shapes seen

    def _room(self, key, ask, like):
        """(pointer, bytes) of the workspace that the handle keeps; ask() says how many bytes calls
        of the sizes `key` need."""
        count = self._sizes.get(key)
        if count is None:
            if len(self._sizes) > 1024:
                self._sizes.clear()
            count = self._sizes[key] = ask()
        if not count:
            return None, 0
        w = self._workspace
        if w is None or w.numel() < count:
            self._workspace = w = self._grown(w, count, like)
        return w.data_ptr(), w.numel()

    def _grown(self, old, count, like):
        """Memory of `count` bytes at least, and twice the old one's: all that is kept is less than
        twice the newest."""
        if old is None:
            return _fresh(count, like)
        new = _fresh(max(count, 2 * old.numel()), like)
        self._replaced.append(old)
        return new


class Rotary(_Handle):
    """Rotary positions with three axes (dcn_rotary): pairs = (time, height, width) pairs of a
    head's channels that turn with each axis; channels past them pass."""

    def __init__(self, ctx: HipDeformConv, head_dim: int, pairs, interleaved: bool = False):
        super().__init__(ctx)
        self.head_dim, self.pairs, self.interleaved = int(head_dim), tuple(int(p) for p in pairs), bool(interleaved)
        _need(len(self.pairs) == 3, "rotary pairs are three numbers (time, height, width)")
        self._freq_shape = (sum(self.pairs),)
        try:
            self._c = {t: _ROTARY.pack(code, self.head_dim, *self.pairs, self.interleaved) for t, code in DTYPES.items()}
        except struct.error:
            raise _outside() from None

    def frequencies(self, base: float = 10000.0, device="cuda"):
        """A usual choice of freq: each axis from 1 down to 1 / base."""
        parts = [base ** (-torch.arange(n, dtype=torch.float64) / max(1, n)) for n in self.pairs]
        return torch.cat(parts).float().to(device)

    def _check(self, positions, freq, tokens, device) -> None:
        _whole("positions", positions, torch.int32, (tokens, 3), device)
        _whole("freq", freq, torch.float32, self._freq_shape, device)

    def run_dev(self, x, positions, freq, out, inverse: bool = False, stream=None) -> None:
        """out = x turned by positions ([tokens][3] int32) times freq; inverse: the gradient."""
        tokens, dtype = _rows("x", x), x.dtype
        heads = x.shape[1]
        shape = (tokens, heads, self.head_dim)
        device = self.ctx.device
        xt, xh, _ = _heads("x", x, dtype, shape, device)
        ot, oh, _ = _heads("out", out, dtype, shape, device)
        self._check(positions, freq, tokens, device)
        _dtype(x)
        status = self._lib.dcn_rotary_dev(
            self._ctx, self._c[dtype], tokens, heads, x.data_ptr(), xt, xh, positions.data_ptr(), freq.data_ptr(),
            inverse, out.data_ptr(), ot, oh, stream and _stream(stream))
        if status:
            self.ctx._check(status)


def _cache(k_pages, v_pages, table, device: int) -> bytes:
    """The packed dcn_cache."""
    if k_pages is None or table is None:
        raise DeformConvError(INVALID_ARGUMENT, "k_pages or table is missing")
    if k_pages.dim() != 4 or table.dim() != 2:
        raise DeformConvError(INVALID_SHAPE, "pages are [pages][page_tokens][heads][channels], the table "
                                             "[sequences][width]")
    shape, dtype = k_pages.shape, k_pages.dtype
    _whole("k_pages", k_pages, dtype, shape, device)
    _whole("v_pages", v_pages, dtype, shape, device)
    _whole("table", table, torch.int32, table.shape, device)
    pages, page_tokens, heads, dim = shape
    try:
        return _CACHE.pack(pages, page_tokens, table.shape[1], heads, dim, _dtype(k_pages))
    except struct.error:
        raise _outside() from None


class CacheAppend(_Handle):
    """Writes new tokens into a paged cache (dcn_cache_append_dev)."""

    def run_dev(self, k, v, k_pages, v_pages, table, cu_q, kv_lens, rotary: Rotary | None = None, positions=None,
                freq=None, q=None, q_out=None, stream=None) -> None:
        """k, v: the new tokens of all sequences, sequence s in rows cu_q[s] .. cu_q[s + 1], the
        last of its kv_lens[s] tokens. Keys are turned by `rotary` on the way, and so is q into
        q_out where it is given."""
        device = self.ctx.device
        cache = _cache(k_pages, v_pages, table, device)
        s, r = self._shape(k, v, table, cu_q, kv_lens, rotary, positions, freq, q, q_out, k_pages.dtype, *k_pages.shape[2:])
        status = self._lib.dcn_cache_append_dev(
            self._ctx, cache, s, r, _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(positions), _ptr(freq), cu_q.data_ptr(),
            kv_lens.data_ptr(), table.data_ptr(), _ptr(q_out), k_pages.data_ptr(), v_pages.data_ptr(),
            stream and _stream(stream))
        if status:
            self.ctx._check(status)

    def run_mx_dev(self, k, v, pages: "MxPages", table, cu_q, kv_lens, rotary: Rotary | None = None, positions=None, freq=None,
                   q=None, q_out=None, stream=None) -> None:
        """run_dev into a microscaled cache (dcn_cache_append_mx_dev); q_out lies on none of q, k and v."""
        if k is None:
            raise DeformConvError(INVALID_ARGUMENT, "k is missing")
        cache = _mx(pages)._pack(table, k.dtype, self.ctx.device)
        s, r = self._shape(k, v, table, cu_q, kv_lens, rotary, positions, freq, q, q_out, k.dtype, pages.kv_heads, pages.head_dim)
        status = self._lib.dcn_cache_append_mx_dev(
            self._ctx, cache, s, r, _ptr(q), k.data_ptr(), v.data_ptr(), _ptr(positions), _ptr(freq), cu_q.data_ptr(),
            kv_lens.data_ptr(), table.data_ptr(), _ptr(q_out), stream and _stream(stream))
        if status:
            self.ctx._check(status)

    def _shape(self, k, v, table, cu_q, kv_lens, rotary, positions, freq, q, q_out, dtype, kv_heads, dim):
        """The packed dcn_append_shape and dcn_rotary (or None), after the checks."""
        device = self.ctx.device
        tokens, sequences = _rows("k", k), table.shape[0]
        shape = (tokens, kv_heads, dim)
        ks, vs = _heads("k", k, dtype, shape, device), _heads("v", v, dtype, shape, device)
        _index("cu_q", cu_q, sequences + 1, device)
        _index("kv_lens", kv_lens, sequences, device)
        q_heads, qs, os = 0, _NO_STRIDES, _NO_STRIDES
        if q is not None:
            _rows("q", q)
            q_heads = q.shape[1]
            shape = (tokens, q_heads, dim)
            _rows("q_out", q_out)
            qs, os = _heads("q", q, dtype, shape, device), _heads("q_out", q_out, dtype, shape, device)
        r = None
        if rotary is not None:
            rotary._check(positions, freq, tokens, device)
            r = rotary._c[dtype]
        try:
            s = _APPEND.pack(sequences, q_heads, tokens, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1])
        except struct.error:
            raise _outside() from None
        return s, r


def _mx(pages) -> "MxPages":
    if not isinstance(pages, MxPages):
        raise DeformConvError(INVALID_ARGUMENT, f"pages is {type(pages).__name__}; expected MxPages")
    return pages


class MxPages:
    """The buffers of a microscaled cache (dcn_pages): blocks of 32 channels are codes of 8 bits (e4m3)
    or 4 (e2m1) and one power of two. k and v are uint8 [pages][kv_heads][page_tokens][head_dim, or
    half of it with 4 bits], k_scales and v_scales uint8 [pages][kv_heads][page_tokens][head_dim / 32]."""

    def __init__(self, k, v, k_scales, v_scales):
        for name, t in (("k", k), ("v", v), ("k_scales", k_scales), ("v_scales", v_scales)):
            if t is None:
                raise DeformConvError(INVALID_ARGUMENT, f"{name} is missing")
            if t.dtype is not torch.uint8:
                raise DeformConvError(INVALID_ARGUMENT, f"{name} is {t.dtype}; expected torch.uint8")
            _need(t.dim() == 4, f"{name} has {t.dim()} dimensions; expected [pages][kv_heads][page_tokens][...]")
        self.head_dim = 32 * k_scales.shape[3]
        _need(self.head_dim > 0 and k.shape[3] in (self.head_dim, self.head_dim // 2),
              f"{k.shape[3]} bytes of codes do not belong to {k_scales.shape[3]} scales")
        self.bits = 8 if k.shape[3] == self.head_dim else 4
        device = k.get_device()
        _whole("v", v, torch.uint8, k.shape, device)
        _whole("k", k, torch.uint8, k.shape, device)
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            _whole(name, t, torch.uint8, k.shape[:3] + (k_scales.shape[3],), device)
        self._buffers, self._device = (k, v, k_scales, v_scales), device
        self.kv_heads, self.page_tokens = k.shape[1], k.shape[2]

    k = property(lambda self: self._buffers[0])
    v = property(lambda self: self._buffers[1])
    k_scales = property(lambda self: self._buffers[2])
    v_scales = property(lambda self: self._buffers[3])

    @classmethod
    def zeros(cls, pages: int, page_tokens: int, kv_heads: int, head_dim: int, bits: int = 8, device="cuda") -> "MxPages":
        _need(bits in (4, 8), f"{bits} bits: a microscaled cache has 8 or 4")
        _need(head_dim > 0 and head_dim % 32 == 0, "a microscaled cache needs a head_dim of whole blocks of 32")
        shape = (pages, kv_heads, page_tokens)
        return cls(*(torch.zeros(*shape, n, dtype=torch.uint8, device=device)
                     for n in (head_dim * bits // 8,) * 2 + (head_dim // 32,) * 2))

    def _pack(self, table, dtype, device: int) -> bytes:
        """The packed dcn_pages of a call with this table."""
        if table is None:
            raise DeformConvError(INVALID_ARGUMENT, "table is missing")
        if table.dim() != 2:
            raise DeformConvError(INVALID_SHAPE, "the table is [sequences][width]")
        _whole("table", table, torch.int32, table.shape, device)
        if self._device != device:
            _on_device("k", self.k, device)
        code = DTYPES.get(dtype)
        if code is None:
            raise DeformConvError(INVALID_ARGUMENT, f"dtype {dtype} is not float16, bfloat16 or float32")
        k, v, k_scales, v_scales = self._buffers
        try:
            return _PAGES.pack(k.shape[0], self.page_tokens, table.shape[1], self.kv_heads, self.head_dim, code, self.bits, 0,
                               k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr())
        except struct.error:
            raise _outside() from None


class CacheRead(_Handle):
    """Reads a microscaled cache back (dcn_cache_read_dev)."""

    def run_dev(self, pages: MxPages, table, cu, kv_lens, k_out, v_out, stream=None) -> None:
        """Rows cu[s] .. cu[s + 1] of k_out and v_out ([tokens][kv_heads][head_dim]) get the last of
        sequence s's kv_lens[s] tokens, rounded to their type."""
        device = self.ctx.device
        tokens, dtype = _rows("k_out", k_out), k_out.dtype
        packed = _mx(pages)._pack(table, dtype, device)
        shape = (tokens, pages.kv_heads, pages.head_dim)
        ks, vs = _heads("k_out", k_out, dtype, shape, device), _heads("v_out", v_out, dtype, shape, device)
        sequences = table.shape[0]
        _index("cu", cu, sequences + 1, device)
        _index("kv_lens", kv_lens, sequences, device)
        try:
            s = _READ.pack(sequences, 0, tokens, ks[0], ks[1], vs[0], vs[1])
        except struct.error:
            raise _outside() from None
        status = self._lib.dcn_cache_read_dev(self._ctx, packed, s, cu.data_ptr(), kv_lens.data_ptr(), table.data_ptr(),
                                              k_out.data_ptr(), v_out.data_ptr(), stream and _stream(stream))
        if status:
            self.ctx._check(status)


class FrameAttention(_Handle):
    """Attention over a window of frames (dcn_attention_shape): a token of frame f sees the
    frames f - back .. f + ahead (negative: without an end) and the first `sinks` ones, frames
    having frame_tokens tokens. frame_tokens = 1 counts in tokens."""

    def __init__(self, ctx: HipDeformConv, q_heads: int, kv_heads: int, head_dim: int, frame_tokens: int = 1,
                 back: int = -1, ahead: int = 0, sinks: int = 0, scale: float | None = None):
        super().__init__(ctx)
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        _need(self.q_heads > 0 and self.kv_heads > 0 and self.q_heads % self.kv_heads == 0,
              "q_heads must be a positive multiple of kv_heads")
        _need(self.head_dim > 0, "head_dim must be positive")
        self.frame_tokens, self.back, self.ahead, self.sinks = int(frame_tokens), int(back), int(ahead), int(sinks)
        self.scale = 1.0 / math.sqrt(self.head_dim) if scale is None else _factor("scale", scale)

    def _pack(self, q, sequences, max_q, max_kv, q_tokens, kv_tokens, *strides) -> bytes:
        """The packed dcn_attention_shape; strides: (token, head, ...) of q, k, v, out, dout, dq, dk, dv."""
        flat = [x for s in strides for x in s[:2]]
        flat += [0] * (16 - len(flat))
        try:
            return _ATTENTION.pack(_dtype(q), sequences, self.q_heads, self.kv_heads, self.head_dim, self.frame_tokens,
                                   self.back, self.ahead, self.sinks, max_q, max_kv, self.scale, q_tokens, kv_tokens, *flat)
        except struct.error:
            raise _outside() from None

    def _runs(self, q_tokens, kv_tokens, cu_q, cu_kv, max_q, max_kv):
        """(sequences, max_q, max_kv): without index arrays, one sequence of all rows, or the
        rows in equal runs of max_q and max_kv."""
        max_q = q_tokens if max_q is None else int(max_q)
        max_kv = kv_tokens if max_kv is None else int(max_kv)
        starts = cu_kv if cu_q is None else cu_q
        if starts is not None:
            if starts.dim() != 1:
                raise DeformConvError(INVALID_SHAPE, f"an index array has {starts.dim()} dimensions; expected one")
            sequences = starts.shape[0] - 1
        else:
            sequences = q_tokens // max_q if max_q else (kv_tokens // max_kv if max_kv else 0)
        if cu_q is not None:
            _index("cu_q", cu_q, sequences + 1, self.ctx.device)
        if cu_kv is not None:
            _index("cu_kv", cu_kv, sequences + 1, self.ctx.device)
        return sequences, max_q, max_kv

    def _forward_parts(self, q, k, v, out, lse, cu_q, cu_kv, max_q, max_kv):
        """What _pack takes, after the checks."""
        q_tokens, kv_tokens, dtype = _rows("q", q), _rows("k", k), q.dtype
        runs = self._runs(q_tokens, kv_tokens, cu_q, cu_kv, max_q, max_kv)
        q_shape, k_shape = (q_tokens, self.q_heads, self.head_dim), (kv_tokens, self.kv_heads, self.head_dim)
        device = self.ctx.device
        strides = (_heads("q", q, dtype, q_shape, device), _heads("k", k, dtype, k_shape, device),
                   _heads("v", v, dtype, k_shape, device), _heads("out", out, dtype, q_shape, device))
        if lse is not None:
            _whole("lse", lse, torch.float32, (q_tokens, self.q_heads), device)
        return (q, *runs, q_tokens, kv_tokens, *strides)

    def _forward_shape(self, q, k, v, out, lse, cu_q, cu_kv, max_q, max_kv) -> _lib.DcnAttentionShape:
        parts = self._forward_parts(q, k, v, out, lse, cu_q, cu_kv, max_q, max_kv)
        return _lib.DcnAttentionShape.from_buffer_copy(self._pack(*parts))

    def _workspace_of(self, s: bytes, which: int, q):
        """The workspace of a call of this shape; strides have no part in its size."""
        return self._room((which, s[:64]), lambda: self._lib.dcn_attention_workspace_bytes(s, which), q)

    def forward_dev(self, q, k, v, out, lse=None, cu_q=None, cu_kv=None, max_q=None, max_kv=None, stream=None) -> None:
        """out = softmax(scale q k^T over what is visible) v; lse ([tokens][q_heads] FP32) is what
        backward_dev reads. cu_q, cu_kv: int32 starts of the sequences and the end of the last;
        max_q and max_kv bound their lengths."""
        s = self._pack(*self._forward_parts(q, k, v, out, lse, cu_q, cu_kv, max_q, max_kv))
        w, size = self._workspace_of(s, PASS_FORWARD, q)
        status = self._lib.dcn_attention_forward_dev(
            self._ctx, s, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(cu_q), _ptr(cu_kv), out.data_ptr(), _ptr(lse), w,
            size, stream and _stream(stream))
        if status:
            self.ctx._check(status)

    def backward_dev(self, q, k, v, out, lse, dout, dq, dk, dv, cu_q=None, cu_kv=None, max_q=None, max_kv=None,
                     stream=None) -> None:
        """The gradients of forward_dev's out, from its arguments, out, lse and dout."""
        parts = self._forward_parts(q, k, v, out, lse, cu_q, cu_kv, max_q, max_kv)
        if lse is None:
            raise DeformConvError(INVALID_ARGUMENT, "lse is missing")
        dtype, q_shape, k_shape, device = q.dtype, q.shape, k.shape, self.ctx.device
        s = self._pack(*parts, _heads("dout", dout, dtype, q_shape, device), _heads("dq", dq, dtype, q_shape, device),
                       _heads("dk", dk, dtype, k_shape, device), _heads("dv", dv, dtype, k_shape, device))
        w, size = self._workspace_of(s, PASS_BACKWARD, q)
        self.ctx._check(self._lib.dcn_attention_backward_dev(
            self.ctx.ctx, s, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            dout.data_ptr(), _ptr(cu_q), _ptr(cu_kv), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), w, size,
            _stream(stream)))

    def paged_dev(self, q, k_pages, v_pages, table, cu_q, kv_lens, out, lse=None, max_q=None, max_kv=None,
                  stream=None) -> None:
        """forward_dev over a paged cache: sequence s has kv_lens[s] keys, its queries being the
        last tokens (one, or a frame's). cu_q None: max_q queries each. max_kv bounds kv_lens
        (default: the table's width)."""
        device = self.ctx.device
        cache = _cache(k_pages, v_pages, table, device)
        sequences, q_tokens, dtype = table.shape[0], _rows("q", q), k_pages.dtype
        if cu_q is not None:
            _index("cu_q", cu_q, sequences + 1, device)
        _index("kv_lens", kv_lens, sequences, device)
        if max_q is None:
            max_q = q_tokens if cu_q is not None else (q_tokens // sequences if sequences else 0)
        if max_kv is None:
            max_kv = table.shape[1] * k_pages.shape[1]
        shape = (q_tokens, self.q_heads, self.head_dim)
        if lse is not None:
            _whole("lse", lse, torch.float32, (q_tokens, self.q_heads), device)
        s = self._pack(q, sequences, int(max_q), int(max_kv), q_tokens, 0, _heads("q", q, dtype, shape, device), _NO_STRIDES,
                       _NO_STRIDES, _heads("out", out, dtype, shape, device))
        w, size = self._workspace_of(s, PASS_PAGED, q)
        status = self._lib.dcn_attention_paged_dev(
            self._ctx, s, cache, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(cu_q), kv_lens.data_ptr(),
            table.data_ptr(), out.data_ptr(), _ptr(lse), w, size, stream and _stream(stream))
        if status:
            self.ctx._check(status)

    def paged_mx_dev(self, q, pages: MxPages, table, cu_q, kv_lens, out, lse=None, max_q=None, max_kv=None, stream=None) -> None:
        """paged_dev over a microscaled cache."""
        if q is None:
            raise DeformConvError(INVALID_ARGUMENT, "q is missing")
        cache = _mx(pages)._pack(table, q.dtype, self.ctx.device)
        self._pages(q, cache, pages.page_tokens, None, table, cu_q, kv_lens, out, lse, max_q, max_kv, stream)

    def shared_dev(self, q, pages, prefix_table, prefix_len, table, cu_q, kv_lens, out, lse=None, max_q=None, max_kv=None,
                   max_prefix=None, stream=None) -> None:
        """paged_dev, or paged_mx_dev, for sequences that share a prefix: prefix_len[0] tokens on the
        pages of prefix_table ([width]) stand before every sequence's own kv_lens[s], of which `table`
        and max_kv speak. pages: an MxPages, or (k_pages, v_pages). Positions, the window and the sinks
        count from the prefix's first token. max_prefix bounds prefix_len (default: the table's width)."""
        device = self.ctx.device
        if q is None:
            raise DeformConvError(INVALID_ARGUMENT, "q is missing")
        if isinstance(pages, MxPages):
            cache, page_tokens = pages._pack(table, q.dtype, device), pages.page_tokens
        else:
            if not isinstance(pages, (tuple, list)) or len(pages) != 2:
                raise DeformConvError(INVALID_ARGUMENT, "pages is neither an MxPages nor (k_pages, v_pages)")
            k_pages, v_pages = pages
            sizes = _cache(k_pages, v_pages, table, device)
            if k_pages.dtype is not q.dtype:
                raise DeformConvError(INVALID_ARGUMENT, f"k_pages is {k_pages.dtype}; expected {q.dtype}")
            cache, page_tokens = sizes + _AS_IS.pack(0, 0, k_pages.data_ptr(), v_pages.data_ptr(), 0, 0), k_pages.shape[1]
        if prefix_table is None:
            raise DeformConvError(INVALID_ARGUMENT, "prefix_table is missing")
        if prefix_table.dim() != 1:
            raise DeformConvError(INVALID_SHAPE, f"prefix_table has {prefix_table.dim()} dimensions; expected one")
        width = prefix_table.shape[0]
        _index("prefix_table", prefix_table, width, device)
        _index("prefix_len", prefix_len, 1, device)
        if max_prefix is None:
            max_prefix = width * page_tokens
        try:
            prefix = _PREFIX.pack(width, int(max_prefix), prefix_table.data_ptr(), prefix_len.data_ptr())
        except struct.error:
            raise _outside() from None
        self._pages(q, cache, page_tokens, prefix, table, cu_q, kv_lens, out, lse, max_q, max_kv, stream)

    def _pages(self, q, cache, page_tokens, prefix, table, cu_q, kv_lens, out, lse, max_q, max_kv, stream) -> None:
        """dcn_attention_pages_dev."""
        device = self.ctx.device
        sequences, q_tokens, dtype = table.shape[0], _rows("q", q), q.dtype
        if cu_q is not None:
            _index("cu_q", cu_q, sequences + 1, device)
        _index("kv_lens", kv_lens, sequences, device)
        if max_q is None:
            max_q = q_tokens if cu_q is not None else (q_tokens // sequences if sequences else 0)
        if max_kv is None:
            max_kv = table.shape[1] * page_tokens
        shape = (q_tokens, self.q_heads, self.head_dim)
        if lse is not None:
            _whole("lse", lse, torch.float32, (q_tokens, self.q_heads), device)
        s = self._pack(q, sequences, int(max_q), int(max_kv), q_tokens, 0, _heads("q", q, dtype, shape, device), _NO_STRIDES,
                       _NO_STRIDES, _heads("out", out, dtype, shape, device))
        # Sizes without pointers and strides: those have no part in the workspace's.
        w, size = self._room((s[:64], cache[:32], prefix and prefix[:8]),
                             lambda: self._lib.dcn_attention_pages_workspace_bytes(s, cache, prefix), q)
        status = self._lib.dcn_attention_pages_dev(
            self._ctx, s, cache, prefix, q.data_ptr(), _ptr(cu_q), kv_lens.data_ptr(), table.data_ptr(), out.data_ptr(),
            _ptr(lse), w, size, stream and _stream(stream))
        if status:
            self.ctx._check(status)


class GatedNorm(_Handle):
    """The norms around a block (dcn_norm_shape): x_out = x + residual_scale * gate * norm(h) *
    w_post, y = norm(x_out) * w_pre, with a row of gates for each run of gate_tokens tokens."""

    def __init__(self, ctx: HipDeformConv, channels: int, gate_tokens: int = 1, residual_scale: float = 1.0,
                 eps: float = 1e-6):
        super().__init__(ctx)
        self.channels, self.gate_tokens = int(channels), int(gate_tokens)
        self.residual_scale, self.eps = _factor("residual_scale", residual_scale), _factor("eps", eps)
        self._kept = None
        self._kept_for = None  # (rstd, packed shape) of the forward that wrote it
        _need(self.channels > 0 and self.gate_tokens > 0, "channels and gate_tokens must be positive")

    def _pack(self, x) -> bytes:
        if x is None:
            raise DeformConvError(INVALID_ARGUMENT, "the residual stream is missing")
        if x.dim() != 2:
            raise DeformConvError(INVALID_SHAPE, f"the residual stream has {x.dim()} dimensions; expected [tokens][channels]")
        try:
            return _NORM.pack(_dtype(x), self.channels, x.shape[0], self.gate_tokens, self.residual_scale, self.eps)
        except struct.error:
            raise _outside() from None

    def _check_all(self, x, needed, tensors, gates, vectors, sums=()) -> None:
        for name, t in needed:
            if t is None:
                raise DeformConvError(INVALID_ARGUMENT, f"{name} is missing")
        tokens, dtype, channels, device = x.shape[0], x.dtype, self.channels, self.ctx.device
        for shape, kind, group in (((tokens, channels), dtype, needed), ((tokens, channels), dtype, tensors),
                                   ((-(-tokens // self.gate_tokens), channels), dtype, gates),
                                   ((channels,), dtype, vectors), ((channels,), torch.float32, sums)):
            for name, t in group:
                if t is not None and not (t.shape == shape and t.dtype is kind and t.is_contiguous() and t.get_device() == device):
                    _whole(name, t, kind, shape, device)

    def low_bytes(self, x) -> int:
        """Bytes of forward_dev's `low` for a residual stream like x."""
        return int(self._lib.dcn_gated_norm_low_bytes(self._pack(x)))

    def _low_of(self, s, low, like):
        """The pointer of the caller's low, checked."""
        if like.dtype is torch.float32:
            return None
        count = self._lib.dcn_gated_norm_low_bytes(s)
        if not count:
            return None
        _on_device("low", low, self.ctx.device)
        if low.dtype != torch.uint8 or low.numel() < count or not low.is_contiguous():
            raise DeformConvError(INVALID_SHAPE, f"low is not {count} adjacent uint8 values")
        return low.data_ptr()

    def _low_to_write(self, s, low, like, rstd):
        """Where a forward that makes rstd writes: the caller's low, or the handle's own."""
        own = self._kept_for
        if low is not None or like.dtype is torch.float32:
            if own is not None and own[0].data_ptr() == rstd.data_ptr():
                self._kept_for = None  # rstd has another forward's now
            return self._low_of(s, low, like)
        self._kept_for = None
        count = self._lib.dcn_gated_norm_low_bytes(s)
        if not count:
            return None
        if self._kept is None or self._kept.numel() < count:
            self._kept = self._grown(self._kept, count, like)
        self._kept_for = (rstd, s)
        return self._kept.data_ptr()

    def _low_to_read(self, s, low, like, rstd):
        """What a backward reads: the caller's low, or the handle's own where the forward that made
        rstd was its last one (the tensor is held, so nothing else can lie there)."""
        if low is not None:
            return self._low_of(s, low, like)
        own = self._kept_for
        if own is None or own[1] != s or own[0].data_ptr() != rstd.data_ptr():
            return None
        return self._kept.data_ptr()

    def forward_dev(self, h, x, gate, w_post, w_pre, x_out, y=None, rstd=None, low=None, stream=None) -> None:
        """gate, w_post, w_pre may be None (ones); y None: no block follows. rstd ([tokens][2]
        FP32) is what backward_dev reads; with it, 16-bit calls keep what rounding takes from
        x_out (low_bytes(x) uint8 values) in `low`, or in the handle until its next such call."""
        s = self._pack(x)
        self._check_all(x, (("h", h), ("x", x), ("x_out", x_out)), (("y", y),), (("gate", gate),),
                        (("w_post", w_post), ("w_pre", w_pre)))
        if rstd is not None:
            _whole("rstd", rstd, torch.float32, (x.shape[0], 2), self.ctx.device)
        status = self._lib.dcn_gated_norm_forward_dev(
            self._ctx, s, h.data_ptr(), x.data_ptr(), _ptr(gate), _ptr(w_post), _ptr(w_pre), x_out.data_ptr(), _ptr(y),
            _ptr(rstd), None if rstd is None else self._low_to_write(s, low, x, rstd), stream and _stream(stream))
        if status:
            self.ctx._check(status)

    def backward_dev(self, h, x_out, gate, w_post, w_pre, rstd, dx_out, dy, dh, dx, dgate=None, dw_post=None,
                     dw_pre=None, low=None, stream=None) -> None:
        """Gradients from those of x_out and y (dy None where y was not made); dgate, dw_post and
        dw_pre (FP32) where they are given. low: that of the forward that made rstd; None: the
        handle's own if that forward was its last with rstd and kept it there, else x_out is
        taken as it was rounded."""
        s = self._pack(x_out)
        self._check_all(x_out, (("h", h), ("x_out", x_out), ("dx_out", dx_out), ("dh", dh), ("dx", dx)),
                        (("dy", dy),), (("gate", gate), ("dgate", dgate)), (("w_post", w_post), ("w_pre", w_pre)),
                        (("dw_post", dw_post), ("dw_pre", dw_pre)))
        _whole("rstd", rstd, torch.float32, (x_out.shape[0], 2), self.ctx.device)
        w, size = self._room(s, lambda: self._lib.dcn_gated_norm_workspace_bytes(s), x_out)
        self.ctx._check(self._lib.dcn_gated_norm_backward_dev(
            self.ctx.ctx, s, h.data_ptr(), x_out.data_ptr(), _ptr(gate), _ptr(w_post), _ptr(w_pre),
            rstd.data_ptr(), self._low_to_read(s, low, x_out, rstd), dx_out.data_ptr(), _ptr(dy), dh.data_ptr(),
            dx.data_ptr(), _ptr(dgate), _ptr(dw_post), _ptr(dw_pre), w, size, _stream(stream)))
