"""What stands between a block's q / k / v projection and its output projection, over the C ABI: the norm and rotation of heads, a cache of
keys and values in eight or four bits, attention of the last tokens over it, and attention of whole prompts.

Heads are [tokens, heads, channels] with the heads of a token beside one another and tokens any distance apart, as `.view(tokens, heads, channels)` of a
projection's output, or of a part of its columns, has them.  Every call goes to the current stream, checks its arguments on the host, and may be captured.
"""
from __future__ import annotations

import ctypes
import math
import struct
from ctypes import c_void_p

import torch

from . import _lib, ops
from ._lib import check
from .ops import _DTYPES, _FLOATS, _given, _load, _refuse, _stream_ptr

_HALVES = (torch.bfloat16, torch.float16)
_PACK_CACHE = struct.Struct("PPPPi4xqqqqffi4x")  # qfg_kv_cache, and the device that it lies on
_IDS = {torch.int32: 4, torch.int64: 8}
# What says in C++ that an object is a cache: a capsule, which nothing but a KvCache makes, of the address of its qfg_kv_cache.
_CAPSULE = b"qfg_kv_cache"
_new_capsule = ctypes.pythonapi.PyCapsule_New
_new_capsule.restype, _new_capsule.argtypes = ctypes.py_object, (c_void_p, ctypes.c_char_p, c_void_p)


def _on_current(t) -> bool:
    return isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == torch.cuda.current_device()


def _heads(op: str, name: str, t, dtypes, dim=None):
    """(tokens, heads, channels, elements from token to token)"""
    if not _on_current(t):
        _refuse(f"{op}: {name} must be a tensor on the current CUDA device")
    if t.dtype not in dtypes:
        _refuse(f"{op}: {name} must be {' / '.join(str(d).removeprefix('torch.') for d in dtypes)}, not {t.dtype}")
    if t.dim() != 3 or t.shape[1] < 1 or t.shape[2] < 1 or (dim is not None and t.shape[2] != dim):
        _refuse(f"{op}: {name} must be [tokens, heads, {'channels' if dim is None else dim}]")
    tokens, heads, n = t.shape
    if tokens == 0:
        return 0, heads, n, heads * n
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != n) or (tokens > 1 and t.stride(0) < heads * n):
        _refuse(f"{op}: the heads of a token of {name} must lie beside one another, and tokens must not overlap")
    return tokens, heads, n, t.stride(0) if tokens > 1 else heads * n


def _whole_numbers(op: str, name: str, t, dtypes, dim: int):
    if not _on_current(t) or t.dtype not in dtypes or t.dim() != dim:
        _refuse(f"{op}: {name} must be a {dim}-D tensor of {' / '.join(str(d).removeprefix('torch.') for d in dtypes)} on the current CUDA device")
    if t.numel() and t.stride(-1) != 1 and t.shape[-1] > 1:
        _refuse(f"{op}: {name} must be contiguous along its last dimension")
    return t


def _table(op: str, table, cache):
    """(address, elements from row to row, sequences, pages of a row)"""
    _whole_numbers(op, "the table", table, (torch.int32,), 2)
    seqs, most = table.shape
    ld = table.stride(0) if seqs > 1 else most
    if seqs > 1 and ld < most:
        _refuse(f"{op}: the rows of the table overlap")
    return table.data_ptr(), ld, seqs, most


def _workspace_bytes(cache, seqs: int, tokens: int, heads: int, most: int) -> int:
    """Of a CacheAttention over `most` pages a sequence; what that refuses of its sizes is refused here."""
    need = ctypes.c_size_t()
    check(_load().qfg_cache_attention_workspace_bytes(cache._at, seqs, tokens, heads, most, ctypes.byref(need)))
    return need.value


class KvCache:
    """Keys and values of all sequences, cut into pages of `page` tokens (a multiple of 32): torch.uint8, block-16 NVFP4 (9/16 of a byte a value), or
    torch.float8_e4m3fn with a scale for each token and head.

    k, v             [pages, kv_heads, page, head_dim] in E4M3, [..., head_dim / 2] in four bits (channel 2 b in the low nibble of byte b)
    k_scale, v_scale [pages, kv_heads, page] FP32, or [pages, kv_heads, page, head_dim / 16] E4M3

    In four bits a stored 1 stands for `k_unit` or `v_unit`, by which values from 2^-10 to 2688 units are held well: a 2688th of the largest value there is
    makes the most of them.  A token's slot is page * (page size) + (its place in the page).  The memory is torch's: new, and zero, or with `of` tensors in hand."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page: int = 64, dtype: torch.dtype = torch.uint8, k_unit: float = 1.0, v_unit: float = 1.0,
                 device="cuda"):
        shape = (int(pages), int(kv_heads), int(page))
        if dtype == torch.uint8:
            kinds = ((head_dim // 2,), torch.uint8), ((head_dim // 16,), torch.float8_e4m3fn)
        elif dtype == torch.float8_e4m3fn:
            kinds = ((head_dim,), torch.float8_e4m3fn), ((), torch.float32)
        else:
            _refuse("KvCache: dtype must be torch.uint8 (block-16 NVFP4) or torch.float8_e4m3fn")
        if min(shape) < 1 or head_dim not in (64, 128, 256) or page % 32 != 0:
            _refuse("KvCache: at least one page and head, pages of a multiple of 32 tokens, heads of 64, 128 or 256 channels")
        self._hold(*[torch.zeros(shape + last, dtype=torch.uint8 if kind == torch.float8_e4m3fn else kind, device=device).view(kind) for _ in range(2)
                     for last, kind in kinds], k_unit, v_unit)

    @classmethod
    def of(cls, k, k_scale, v, v_scale, k_unit: float = 1.0, v_unit: float = 1.0) -> "KvCache":
        """A cache over tensors in hand."""
        cache = cls.__new__(cls)
        cache._hold(k, k_scale, v, v_scale, k_unit, v_unit)
        return cache

    def _hold(self, k, k_scale, v, v_scale, k_unit, v_unit):
        if not all(isinstance(t, torch.Tensor) and t.is_cuda and t.is_contiguous() for t in (k, k_scale, v, v_scale)):
            _refuse("KvCache: keys, values and their scales must be contiguous CUDA tensors")
        if k.dim() != 4 or k.dtype not in (torch.uint8, torch.float8_e4m3fn) or v.shape != k.shape or v.dtype != k.dtype:
            _refuse("KvCache: keys and values must be [pages, kv_heads, page, channels], of torch.uint8 or torch.float8_e4m3fn")
        fp4 = k.dtype == torch.uint8
        dim = k.shape[3] * 2 if fp4 else k.shape[3]
        shape, kind = (k.shape[:3] + (dim // 16,), torch.float8_e4m3fn) if fp4 else (k.shape[:3], torch.float32)
        if any(t.shape != shape or t.dtype != kind for t in (k_scale, v_scale)):
            _refuse(f"KvCache: the scales must be {str(kind).removeprefix('torch.')} {list(shape)}")
        if len({t.get_device() for t in (k, k_scale, v, v_scale)}) != 1:
            _refuse("KvCache: all tensors must be on one device")
        if dim not in (64, 128, 256) or k.shape[2] % 32 != 0 or min(k.shape) < 1:
            _refuse("KvCache: at least one page and head, pages of a multiple of 32 tokens, heads of 64, 128 or 256 channels")
        if not all(1e-18 <= float(u) <= 1e18 for u in (k_unit, v_unit)):
            _refuse("KvCache: the units must lie between 1e-18 and 1e18")
        if any(t.data_ptr() % 16 for t in (k, k_scale, v, v_scale)):
            _refuse("KvCache: the tensors must begin on 16 bytes")
        self._k, self._k_scale, self._v, self._v_scale = k, k_scale, v, v_scale
        self.pages, self.kv_heads, self.page, self.head_dim = k.shape[0], k.shape[1], k.shape[2], dim
        self.dtype, self.k_unit, self.v_unit = k.dtype, float(k_unit), float(v_unit)
        self._packed = ctypes.create_string_buffer(_PACK_CACHE.pack(k.data_ptr(), k_scale.data_ptr(), v.data_ptr(), v_scale.data_ptr(), _DTYPES[k.dtype],
                                                                    self.pages, self.kv_heads, self.page, dim, self.k_unit, self.v_unit, k.get_device()))
        self._at = ctypes.addressof(self._packed)
        self._capsule = _new_capsule(self._at, _CAPSULE, None)

    k = property(lambda self: self._k)
    k_scale = property(lambda self: self._k_scale)
    v = property(lambda self: self._v)
    v_scale = property(lambda self: self._v_scale)


def _cache(op: str, cache) -> int:
    if not isinstance(cache, KvCache):
        _refuse(f"{op}: the cache must be a KvCache")
    if cache._k.get_device() != torch.cuda.current_device():
        _refuse(f"{op}: the cache must be on the current CUDA device")
    return cache._at


class QkNormRope:
    """Norm of each query and key head, rotation by position, and, with a cache, the write of keys and values, in one pass.

    y = x * rsqrt(mean(x^2) + eps) * (weight_offset + weight) over a head's channels (no weight: y = x); then pairs of the first `rotary_dim` channels turn by
    position * inv_freq[pair]: (i, i + rotary_dim / 2), or neighbours if `interleaved`; the others stay.  FP32 throughout, rounded once.

    head_dim     64, 128 or 256; rotary_dim a multiple of 32 up to it (all of it unless given; 0: no rotation)
    inv_freq     the pairs' frequencies in radians a position; unless given base^(-2 i / rotary_dim)
    sections     of several axes (time, height, width): how many pairs go by each, in order; or `axes`, the axis of each pair
    rotary_scale a factor of sine and cosine

    (q, k, positions, q_weight, k_weight) -> (q, k), rotated; with v, cache and slots -> q alone, or with keys=True (q, k), keys and values being in the cache."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0, inv_freq=None, sections=None, axes=None, interleaved: bool = False,
                 eps: float = 1e-6, weight_offset: float = 0.0, rotary_scale: float = 1.0):
        lib = _load()
        self._lib, self._h, self._p = lib, c_void_p(), None
        rotary = head_dim if rotary_dim is None else int(rotary_dim)
        pairs = rotary // 2
        if head_dim not in (64, 128, 256) or rotary < 0 or rotary > head_dim or rotary % 32 != 0:
            _refuse("QkNormRope: heads have 64, 128 or 256 channels, of which a multiple of 32 is rotated")
        if inv_freq is None:
            if not float(base) > 0.0:
                _refuse("QkNormRope: the base must be positive")
            inv_freq = [float(base) ** (-i / pairs) for i in range(pairs)]
        inv_freq = [float(f) for f in inv_freq]
        if sections is not None and axes is not None:
            _refuse("QkNormRope: give sections or axes")
        if sections is not None:
            axes = [a for a, n in enumerate(sections) for _ in range(int(n))]
        axes = [0] * pairs if axes is None else [int(a) for a in axes]
        if len(inv_freq) != pairs or len(axes) != pairs:
            _refuse(f"QkNormRope: there must be a frequency and an axis for each of {pairs} pairs")
        self._read = max(axes, default=0) + 1  # rows of positions that any pair goes by are among so many
        self.head_dim, self.rotary_dim, self.axes = head_dim, rotary, max(self._read, len(sections) if sections is not None else 0)
        check(lib.qfg_qk_norm_rope_create((ctypes.c_double * max(1, pairs))(*inv_freq), (ctypes.c_int32 * max(1, pairs))(*axes), pairs, head_dim, int(bool(interleaved)),
                                          float(rotary_scale), float(eps), float(weight_offset), ctypes.byref(self._h)))
        self._p = self._h.value

    def __call__(self, q, k, positions=None, q_weight=None, k_weight=None, v=None, cache: KvCache | None = None, slots=None, keys: bool = False):
        """positions [tokens], or [axes, tokens] of as many as `sections` has, int64 or int32; slots [tokens] int64: a token whose slot is negative or lies
        behind the cache is not written; slots must differ."""
        if self.axes > self._read and self.rotary_dim:  # the last sections have no pairs
            if not isinstance(positions, torch.Tensor) or positions.dim() != 2 or positions.shape[0] != self.axes:
                _refuse(f"QkNormRope: positions must be [{self.axes}, tokens]")
            positions = positions[:self._read]
        r = ops._calls.qk_norm_rope(self._p, q, k, positions, q_weight, k_weight, v, cache._capsule if cache.__class__ is KvCache else cache, slots, keys)
        if r is not None:
            return r if r.__class__ is not int else check(r)
        op = "QkNormRope"
        tokens, q_heads, dim, ldq = _heads(op, "q", q, _FLOATS, self.head_dim)
        of, kv_heads, _, ldk = _heads(op, "k", k, (q.dtype,), dim)
        if of != tokens:
            _refuse(f"{op}: q and k must have as many tokens")
        where, wide, ldp, axes = None, 8, 0, self._read
        if self.rotary_dim:
            if positions is None:
                _refuse(f"{op}: no positions")
            p = positions.unsqueeze(0) if isinstance(positions, torch.Tensor) and positions.dim() == 1 else positions
            _whole_numbers(op, "positions", p, tuple(_IDS), 2)
            if tuple(p.shape) != (axes, tokens):
                _refuse(f"{op}: positions must be [{tokens}]" if self.axes == 1 else f"{op}: positions must be [{self.axes}, {tokens}]")
            if axes > 1 and tokens > 0 and p.stride(0) < tokens:
                _refuse(f"{op}: the axes of positions overlap")
            where, wide, ldp = p.data_ptr(), _IDS[p.dtype], p.stride(0) if axes > 1 else tokens
        kind = q.dtype
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is None:
                continue
            if not _on_current(w) or w.dtype not in (q.dtype, torch.float32) or tuple(w.shape) != (dim,) or not w.is_contiguous():
                _refuse(f"{op}: {name} must be a contiguous tensor of {dim} elements, of the type of q or FP32")
            kind = w.dtype
        if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
            _refuse(f"{op}: both weights must be of one type")
        at = vp = sp = None
        ldv = 0
        if cache is not None:
            at = _cache(op, cache)
            of, heads, _, ldv = _heads(op, "v", v, (q.dtype,), dim)
            _whole_numbers(op, "slots", slots, (torch.int64,), 1)
            if (of, heads) != (tokens, kv_heads) or slots.shape[0] != tokens or (cache.kv_heads, cache.head_dim) != (kv_heads, dim):
                _refuse(f"{op}: v, the slots and the cache must fit k")
            vp, sp = v.data_ptr(), slots.data_ptr()
        elif v is not None or slots is not None:
            _refuse(f"{op}: v and slots go with a cache")
        q_out = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=q.device)
        k_out = torch.empty((tokens, kv_heads, dim), dtype=q.dtype, device=q.device) if cache is None or keys else None
        check(self._lib.qfg_qk_norm_rope_compute(self._p, _DTYPES[q.dtype], q.data_ptr(), ldq, q_heads, k.data_ptr(), ldk, kv_heads, vp, ldv, where, wide, ldp, axes,
                                                 q_weight.data_ptr() if q_weight is not None else None, k_weight.data_ptr() if k_weight is not None else None,
                                                 _DTYPES[kind], tokens, q_out.data_ptr(), k_out.data_ptr() if k_out is not None else None, at, sp, _stream_ptr()))
        return q_out if k_out is None else (q_out, k_out)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            self._lib.qfg_qk_norm_rope_destroy(h)
            self._h = self._p = None


class CacheWrite:
    """(k, v, cache, slots): keys and values [tokens, kv_heads, head_dim] in BF16, FP16 or FP32, as they are, into their slots of a KvCache.  A token whose slot
    (int64) is negative or lies behind the cache is not written; slots must differ."""

    def __init__(self):
        self._lib = _load()

    def __call__(self, k, v, cache: KvCache, slots) -> None:
        r = ops._calls.cache_write(k, v, cache._capsule if cache.__class__ is KvCache else cache, slots)
        if r is not None:
            return check(r)
        op = "CacheWrite"
        at = _cache(op, cache)
        tokens, heads, _, ldk = _heads(op, "k", k, _FLOATS, cache.head_dim)
        of, also, _, ldv = _heads(op, "v", v, (k.dtype,), cache.head_dim)
        _whole_numbers(op, "slots", slots, (torch.int64,), 1)
        if (of, also) != (tokens, heads) or heads != cache.kv_heads or slots.shape[0] != tokens:
            _refuse(f"{op}: k, v, the slots and the cache must fit one another")
        check(self._lib.qfg_cache_write(_DTYPES[k.dtype], k.data_ptr(), ldk, v.data_ptr(), ldv, tokens, at, slots.data_ptr(), _stream_ptr()))


class CacheRead:
    """(cache, table, offsets, rows) -> (k, v) [rows, kv_heads, head_dim] in `dtype`: rows offsets[i] to offsets[i + 1] are the first tokens of sequence i, whose
    pages are table[i] (int32 [sequences, most pages]); offsets int32 [sequences + 1].  Rows of no sequence are left as they were (`out`; new tensors hold
    anything there); tokens that no page of the cache holds become zeros."""

    def __init__(self, dtype: torch.dtype = torch.bfloat16):
        self._lib = _load()
        if dtype not in _FLOATS:
            _refuse("CacheRead: dtype must be torch.bfloat16, torch.float16 or torch.float32")
        self.dtype, self._code = dtype, _DTYPES[dtype]

    def __call__(self, cache: KvCache, table, offsets, rows: int, out=None):
        if out is None:
            r = ops._calls.cache_read(self._code, cache._capsule if cache.__class__ is KvCache else cache, table, offsets, rows)
            if r is not None:
                return r if r.__class__ is tuple else check(r)
        op = "CacheRead"
        at = _cache(op, cache)
        tp, ldt, seqs, most = _table(op, table, cache)
        _whole_numbers(op, "offsets", offsets, (torch.int32,), 1)
        if offsets.shape[0] != seqs + 1 or int(rows) < 0:
            _refuse(f"{op}: there must be {seqs + 1} offsets, and no fewer than 0 rows")
        shape = (int(rows), cache.kv_heads, cache.head_dim)
        if out is None:
            out = tuple(torch.empty(shape, dtype=self.dtype, device=table.device) for _ in range(2))
        if len(out) != 2:
            _refuse(f"{op}: out must be (k, v)")
        k, v = (_given(op, name, t, shape, self.dtype) for name, t in zip("kv", out))
        check(self._lib.qfg_cache_read(at, tp, ldt, seqs, most, offsets.data_ptr(), int(rows), self._code, k.data_ptr(), v.data_ptr(), _stream_ptr()))
        return k, v


def _scale(op: str, scale):
    if scale is not None and not 0.0 < float(scale) <= 1e18:
        _refuse(f"{op}: the scale must be positive and finite")
    return 0.0 if scale is None else float(scale)


class CacheAttention:
    """softmax(scale q k^T) v of the last tokens of each sequence over its tokens in a KvCache.

    q [sequences, tokens, heads, head_dim] (or, of one token each, [sequences, heads, head_dim]) in BF16 or FP16; table int32 [sequences, most pages]: each
    sequence's pages; lengths int32 [sequences]: its tokens in the cache, those of q among them.  Token t sees the first lengths - tokens + 1 + t of them;
    a row that sees nothing is 0; a value within a sequence that is not finite makes the rows of its key head NaN.  Query head h reads key head
    h // (heads // kv_heads).  `scale`: 1 / sqrt(head_dim) unless given.  Returns a tensor like q; with
    lse=True also the logarithm of each row's sum of exponentials, FP32, by which attention over several caches can be joined.  A call allocates its own workspace."""

    def __init__(self, scale: float | None = None):
        self._lib = _load()
        self.scale = _scale("CacheAttention", scale)

    def __call__(self, q, cache: KvCache, table, lengths, out=None, lse: bool = False):
        if out is None:
            r = ops._calls.cache_attention(self.scale, q, cache._capsule if cache.__class__ is KvCache else cache, table, lengths, lse)
            if r is not None:
                return r if r.__class__ is not int else check(r)
        op = "CacheAttention"
        at = _cache(op, cache)
        if not _on_current(q) or q.dtype not in _HALVES or q.dim() not in (3, 4) or q.shape[-1] != cache.head_dim or q.shape[-2] < 1:
            _refuse(f"{op}: q must be [sequences, tokens, heads, {cache.head_dim}] in BF16 or FP16 on the current CUDA device")
        four = q.unsqueeze(1) if q.dim() == 3 else q
        seqs, tokens, heads, dim = four.shape
        if q.numel() and (four.stride(3) != 1 or (heads > 1 and four.stride(2) != dim)):
            _refuse(f"{op}: the heads of a token of q must lie beside one another")
        ld_token = four.stride(1) if tokens > 1 else heads * dim
        ld_seq = four.stride(0) if seqs > 1 else tokens * heads * dim
        tp, ldt, of, most = _table(op, table, cache)
        _whole_numbers(op, "lengths", lengths, (torch.int32,), 1)
        if of != seqs or lengths.shape[0] != seqs:
            _refuse(f"{op}: there must be a row of the table and a length for each of {seqs} sequences")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _given(op, "out", out, q.shape, q.dtype)
        sums = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if lse else None
        need = _workspace_bytes(cache, seqs, tokens, heads, most)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        check(self._lib.qfg_cache_attention(_DTYPES[q.dtype], q.data_ptr(), ld_seq, ld_token, seqs, tokens, heads, at, tp, ldt, most, lengths.data_ptr(),
                                            self.scale or 1 / math.sqrt(dim), workspace.data_ptr() if workspace is not None else None, out.data_ptr(),
                                            sums.data_ptr() if lse else None, _stream_ptr()))
        return (out, sums) if lse else out


class PromptAttention:
    """softmax(scale q k^T) v of packed sequences of different lengths.

    q [rows, heads, head_dim], k and v [key rows, kv_heads, head_dim] in BF16 or FP16, heads of 64 or 128 channels; rows q_offsets[i] to q_offsets[i + 1]
    (int32 [sequences + 1]) attend to key rows k_offsets[i] to k_offsets[i + 1] (the same ones unless given).  Causal: the last query of a sequence sees all of
    its keys, each one ahead of it one fewer.  A row that sees nothing is 0; rows of no sequence are left as they were (`out`; a new tensor holds anything
    there).  `scale`: 1 / sqrt(head_dim) unless given.  Returns [rows, heads, head_dim]; with lse=True also the logarithm of each row's sum of exponentials, FP32.

    What lies in the keys and values of other sequences takes no part, whatever it is.  Within a sequence, a value that is not finite makes rows of its head
    up to 128 tokens ahead of it NaN as well.  A row that has a score of NaN or +infinity is NaN.  Scores (scale q k) have to stay below 2^28: a row whose
    largest is further from 0 than that may become NaN."""

    def __init__(self, scale: float | None = None, causal: bool = True):
        self._lib = _load()
        self.scale, self.causal = _scale("PromptAttention", scale), bool(causal)

    def __call__(self, q, k, v, q_offsets, k_offsets=None, out=None, lse: bool = False):
        if out is None:
            r = ops._calls.prompt_attention(self.scale, self.causal, q, k, v, q_offsets, k_offsets, lse)
            if r is not None:
                return r if r.__class__ is not int else check(r)
        op = "PromptAttention"
        rows, heads, dim, ldq = _heads(op, "q", q, _HALVES)
        k_rows, kv_heads, _, ldk = _heads(op, "k", k, (q.dtype,), dim)
        of, also, _, ldv = _heads(op, "v", v, (q.dtype,), dim)
        if (of, also) != (k_rows, kv_heads):
            _refuse(f"{op}: k and v must have the same tokens and heads")
        if k_offsets is None:
            k_offsets = q_offsets
        for name, t in (("q_offsets", q_offsets), ("k_offsets", k_offsets)):
            _whole_numbers(op, name, t, (torch.int32,), 1)
        if q_offsets.shape[0] < 1 or q_offsets.shape != k_offsets.shape:
            _refuse(f"{op}: there must be one offset more than sequences, of queries and of keys")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        _given(op, "out", out, q.shape, q.dtype)
        sums = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if lse else None
        check(self._lib.qfg_prompt_attention(_DTYPES[q.dtype], q.data_ptr(), ldq, rows, heads, k.data_ptr(), ldk, v.data_ptr(), ldv, k_rows, kv_heads, dim,
                                             q_offsets.data_ptr(), k_offsets.data_ptr(), q_offsets.shape[0] - 1, int(self.causal),
                                             self.scale or 1 / math.sqrt(dim), out.data_ptr(), sums.data_ptr() if lse else None, _stream_ptr()))
        return (out, sums) if lse else out
