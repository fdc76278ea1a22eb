"""The keys and values of many requests in a paged cache on the device (KvCache), and what runs between a block's q/k/v and output
projections: new tokens into the cache with the rotation of keys and queries by their positions (Rope, kv_append), attention over the
pages (attend) and over a few pages for each row (attend_selected).

Calls describe their requests by row_offsets [requests + 1], lengths [requests] and tables [requests][width], all int32: request r's new
tokens are rows row_offsets[r] .. row_offsets[r + 1] - 1, the last of its lengths[r] tokens, whose page i is tables[r][i]. As for the
projections, numpy arrays use the synchronous host entry points and torch GPU tensors the ``_dev`` ones; the cache lies on the device either
way. The Context.bind_*_dev methods convert a call's arguments once.
"""
import ctypes
import math

import numpy as np

from . import _lib
from .errors import (OverfitArgumentError, OverfitArgumentNullError, OverfitArgumentOutOfRangeError, OverfitUnsupportedTypeError,
                     raise_for_status)
from .runtime import BoundCall, as_buf, default_context, same_side, torch
from .step import _context, _empty, _ptr, _sized

_TYPES = {_lib.TYPE_F16: "float16", _lib.TYPE_BF16: "bfloat16", _lib.TYPE_I8: "uint8"}
PAGE_SIZES = (32, 64, 128, 256)


class _DeviceBytes:
    """A stretch of a cache's device memory for torch to wrap; keeps the cache alive."""

    def __init__(self, cache, address, count, typestr):
        self._cache = cache
        self.__cuda_array_interface__ = {"shape": (count,), "typestr": typestr, "data": (address, False), "version": 2}


class KvCache:
    """`pages` pages of `page_size` tokens (32, 64, 128 or 256) of `kv_heads` heads of `head_dim` channels (ovfq_kv_create), kept in
    `type_id`: TYPE_F16, TYPE_BF16 or TYPE_I8. sums: each full page's sum of keys is kept too, for attend_selected."""

    def __init__(self, kv_heads: int, head_dim: int, page_size: int, pages: int, type_id=_lib.TYPE_F16, sums=False, ctx=None):
        if type_id not in _TYPES:
            raise OverfitUnsupportedTypeError(f"cache type {type_id}")
        if not 1 <= kv_heads <= _lib.MAX_KV_HEADS:
            raise OverfitArgumentOutOfRangeError(f"kv_heads ({kv_heads}) must be in [1, {_lib.MAX_KV_HEADS}]")
        if not 1 <= head_dim <= _lib.MAX_HEAD_DIM:
            raise OverfitArgumentOutOfRangeError(f"head_dim ({head_dim}) must be in [8, {_lib.MAX_HEAD_DIM}]")
        if head_dim % 8:
            raise OverfitArgumentError(f"head_dim ({head_dim}) must be a multiple of 8")
        if page_size not in PAGE_SIZES:
            raise OverfitArgumentOutOfRangeError(f"page_size ({page_size}) must be one of {PAGE_SIZES}")
        if pages < 1:
            raise OverfitArgumentOutOfRangeError(f"pages ({pages}) must be positive")
        if pages * page_size >= 1 << 31:
            raise OverfitArgumentError(f"{pages} pages of {page_size} tokens exceed 2^31 - 1")
        self._ctx = ctx or default_context()
        h = ctypes.c_void_p()
        raise_for_status(self._ctx.lib.ovfq_kv_create(self._ctx.handle, type_id, kv_heads, head_dim, page_size, pages, int(bool(sums)),
                                                      ctypes.byref(h)), self._ctx.lib)
        self.handle = h
        self.kv_heads, self.head_dim, self.page_size, self.pages, self.type_id = kv_heads, head_dim, page_size, pages, type_id
        self.sums = bool(sums)

    def __del__(self):
        h = getattr(self, "handle", None)
        if h is not None and h.value:
            try:
                self._ctx.lib.ovfq_kv_destroy(h)
            except Exception:
                pass
            self.handle = None

    @property
    def context(self):
        return self._ctx

    def _info(self):
        dp, n, mem, sums = ctypes.c_int(), ctypes.c_size_t(), ctypes.c_void_p(), ctypes.c_void_p()
        raise_for_status(self._ctx.lib.ovfq_kv_info(self.handle, None, None, None, None, None, ctypes.byref(dp), ctypes.byref(n),
                                                    ctypes.byref(mem), ctypes.byref(sums)), self._ctx.lib)
        return dp.value, n.value, mem.value, sums.value

    @property
    def byte_count(self) -> int:
        return self._info()[1]

    def _wrap(self, address, count, typestr):
        return torch.as_tensor(_DeviceBytes(self, address, count, typestr), device=f"cuda:{self._ctx.device}")

    def _view(self, sizes, strides, at):
        """Elements of the cache's type at byte `at` of every block: [pages][page / 32], `sizes` with `strides` up to the heads' place,
        kv_heads, the rest."""
        dp, _, mem, _ = self._info()
        i8 = self.type_id == _lib.TYPE_I8
        each = 1 if i8 else 2
        block, blocks = dp * 64 * each + (256 if i8 else 0), self.page_size // 32
        total = self.pages * self.kv_heads * blocks * block
        t = self._wrap(mem, total, "|u1")
        t = t if i8 else t.view(getattr(torch, _TYPES[self.type_id]))
        e = block // each
        tokens, channels = sizes
        return t.as_strided((self.pages, blocks, *tokens, self.kv_heads, *channels),
                            (e * blocks * self.kv_heads, e, *strides[0], e * blocks, *strides[1]), at // each)

    def key_view(self):
        """The stored keys as a view of the cache's memory: [pages][page_size / 32][2][16][kv_heads][channels / 32][4][8], which read in
        order are [pages][page_size][kv_heads][channels] (channels: head_dim rounded up, zeros behind it). TYPE_I8 caches give
        quants + 128, with their channels as [channels / 64][2][4][8]."""
        dp = self._info()[0]
        if self.type_id == _lib.TYPE_I8:
            return self._view(((2, 16), (dp // 64, 2, 4, 8)), ((dp * 16, 16), (1024, 8, 256, 1)), 0)
        return self._view(((2, 16), (dp // 32, 4, 8)), ((dp * 16, 8), (512, 128, 1)), 0)

    def value_view(self):
        """The stored values likewise: [pages][page_size / 32][2][4][4][kv_heads][channels / 16][16] (TYPE_I8: [channels / 32][2][16])."""
        dp = self._info()[0]
        if self.type_id == _lib.TYPE_I8:
            return self._view(((2, 4, 4), (dp // 32, 2, 16)), ((4, 256, 1), (1024, 8, 16)), dp * 32)
        return self._view(((2, 4, 4), (dp // 16, 16)), ((4, 128, 1), (512, 8)), dp * 64)

    def scale_view(self):
        """TYPE_I8: the scales, [pages][page_size / 32][2 (keys, values)][32][kv_heads]."""
        if self.type_id != _lib.TYPE_I8:
            raise OverfitUnsupportedTypeError("only TYPE_I8 caches have scales")
        dp, _, mem, _ = self._info()
        block, blocks = (dp * 64 + 256) // 4, self.page_size // 32
        t = self._wrap(mem, self.pages * self.kv_heads * blocks * block, "<f4")
        return t.as_strided((self.pages, blocks, 2, 32, self.kv_heads), (block * blocks * self.kv_heads, block, 32, 1, block * blocks),
                            dp * 16)

    def sum_view(self):
        """The pages' sums of keys, [pages][kv_heads][head_dim], each as of when its page was last filled."""
        address = self._info()[3]
        if not address:
            raise OverfitArgumentError("the cache keeps no sums of its pages")
        return self._wrap(address, self.pages * self.kv_heads * self.head_dim, "<f4").view(self.pages, self.kv_heads, self.head_dim)


class Rope:
    """Rotary positions (ovfq_rope): inv_freq [rotary_dim / 2], style "pairs" (channels 2 j and 2 j + 1) or "halves" (j and
    j + rotary_dim / 2), a factor `scale` on cosines and sines, and with several axes of positions pair_axes [rotary_dim / 2] (int32)."""

    __slots__ = ("inv_freq", "style", "scale", "pair_axes")
    STYLES = {"pairs": 0, "halves": 1}

    def __init__(self, inv_freq, style="pairs", scale=1.0, pair_axes=None):
        if style not in self.STYLES:
            raise OverfitArgumentError(f"rope style must be one of {sorted(self.STYLES)}, not {style!r}")
        if not math.isfinite(scale):
            raise OverfitArgumentOutOfRangeError(f"scale ({scale}) must be finite")
        if inv_freq is None:
            raise OverfitArgumentNullError("inv_freq is None")
        self.inv_freq, self.style, self.scale, self.pair_axes = inv_freq, style, float(scale), pair_axes


def _rows_of(x, width, name):
    """Rows of a plane of `width` values each."""
    if x.size == 0 or x.size % width:
        raise OverfitArgumentError(f"{name} has {x.size} elements, not whole rows of {width}")
    return x.size // width


def _query_rows(q, qb, rows, requests, dim):
    """Rows of a plane of queries: the given number, or its first axis ([rows][heads * dim] or [rows][heads][dim]); a plane of one axis is one
    row's, so of one request."""
    axes = len(q.shape)
    if rows is None:
        if axes == 1 and requests > 1:
            raise OverfitArgumentError(f"q of one axis beside {requests} requests: give rows")
        if axes > 3 or (axes == 3 and q.shape[2] != dim):
            raise OverfitArgumentError(f"q of shape {tuple(q.shape)} is neither [rows][heads * {dim}] nor [rows][heads][{dim}]: give rows")
        rows = int(q.shape[0]) if axes > 1 else 1
    if rows <= 0 or qb.size == 0 or qb.size % (rows * dim):
        raise OverfitArgumentError(f"q has {qb.size} elements, not whole heads of {dim} for each of {rows} rows")
    return rows


def _overlap(a, b):
    """Whether two planes of 32-bit values share memory."""
    return a is not None and b is not None and a.ptr < b.ptr + 4 * b.size and b.ptr < a.ptr + 4 * a.size


def _apart(name, written, **others):
    """Refuses an output that shares memory with what the call reads or writes besides."""
    for other, b in others.items():
        if _overlap(written, b):
            raise OverfitArgumentError(f"{name} overlaps {other}")


def _batch(row_offsets, lengths, tables, max_rows):
    """(ovfq_kv_batch, its buffers)."""
    ob = as_buf(row_offsets, np.int32, "row_offsets")
    lb = as_buf(lengths, np.int32, "lengths")
    tb = as_buf(tables, np.int32, "tables")
    requests = ob.size - 1
    if requests < 1:
        raise OverfitArgumentError("row_offsets needs an entry for each request and one more")
    _sized(lb, requests, "lengths")
    if tb.size == 0 or tb.size % requests:
        raise OverfitArgumentError(f"tables has {tb.size} entries, not as many for each of {requests} requests")
    if max_rows < 0:
        raise OverfitArgumentOutOfRangeError(f"max_rows ({max_rows}) must not be negative")
    return _lib.KvBatchStruct(requests, tb.size // requests, max_rows, ob.ptr, lb.ptr, tb.ptr), [ob, lb, tb]


def _call(cache, ctx, name, side, args, keep):
    if ctx is not None and ctx is not cache.context:
        raise OverfitArgumentError("the cache belongs to another context")
    dev = same_side(*side)
    ctx = _context(cache.context, side)
    fn = getattr(ctx.lib, name + "_dev" if dev else name)
    return BoundCall(ctx, fn, (ctx.handle, cache.handle, *args), (cache, side, keep))


def _append_call(cache, k, v, row_offsets, lengths, tables, q, q_out, rope, positions, max_rows, rows=None, ctx=None):
    batch, side = _batch(row_offsets, lengths, tables, max_rows)
    kb, vb = as_buf(k, np.float32, "k", allow_none=True), as_buf(v, np.float32, "v", allow_none=True)
    qb = as_buf(q, np.float32, "q", allow_none=True)
    if (kb is None) != (vb is None):
        raise OverfitArgumentNullError("k and v go together")
    if kb is None and qb is None:
        raise OverfitArgumentNullError("k, v and q are None")
    if kb is not None:
        of_keys = _rows_of(kb, cache.kv_heads * cache.head_dim, "k")
        if vb.size != kb.size:
            raise OverfitArgumentError(f"k has {kb.size} elements, v {vb.size}")
        if rows not in (None, of_keys):
            raise OverfitArgumentError(f"k has {of_keys} rows, not {rows}")
        rows = of_keys
    heads = 0
    if qb is not None:
        if rope is None:
            raise OverfitArgumentNullError("q without a rope")
        rows = _query_rows(q, qb, rows, batch.requests, cache.head_dim)
        heads = qb.size // (rows * cache.head_dim)
        if heads % cache.kv_heads:
            raise OverfitArgumentError(f"heads ({heads}) must be a multiple of kv_heads ({cache.kv_heads})")
        if q_out is None:
            q_out = _empty(qb, qb.size).reshape(tuple(q.shape))
    elif q_out is not None:
        raise OverfitArgumentNullError("q_out without q")
    yb = _sized(as_buf(q_out, np.float32, "q_out", allow_none=True), rows * heads * cache.head_dim, "q_out")
    ob, lb, tb = side
    _apart("q_out", yb, k=kb, v=vb, q=None if yb is not None and yb.ptr == qb.ptr else qb, row_offsets=ob, lengths=lb, tables=tb)
    side += [kb, vb, qb, yb]
    rs = pb = None
    if rope is not None:
        if not isinstance(rope, Rope):
            raise OverfitArgumentError("rope must be a Rope")
        fb = as_buf(rope.inv_freq, np.float32, "inv_freq")
        if fb.size == 0 or 2 * fb.size > cache.head_dim:
            raise OverfitArgumentOutOfRangeError(f"inv_freq has {fb.size} entries: 1 to {cache.head_dim // 2} are taken")
        pb = as_buf(positions, np.int32, "positions", allow_none=True)
        axes = 1
        if pb is not None:
            axes = _rows_of(pb, rows, "positions")
            if axes > _lib.MAX_ROPE_AXES:
                raise OverfitArgumentOutOfRangeError(f"positions of {axes} axes: at most {_lib.MAX_ROPE_AXES} are taken")
        xb = _sized(as_buf(rope.pair_axes, np.int32, "pair_axes", allow_none=True), fb.size, "pair_axes")
        if pb is None and xb is not None:
            axes = _lib.MAX_ROPE_AXES  # every axis has the token's place
        _apart("q_out", yb, inv_freq=fb, positions=pb, pair_axes=xb)
        side += [fb, pb, xb]
        rs = _lib.RopeStruct(2 * fb.size, Rope.STYLES[rope.style], axes, rope.scale, fb.ptr, _ptr(xb))
    elif positions is not None:
        raise OverfitArgumentNullError("positions without a rope")
    args = (ctypes.byref(batch), _ptr(kb), _ptr(vb), rows, None if rs is None else ctypes.byref(rs), _ptr(pb), _ptr(qb), heads, _ptr(yb))
    return _call(cache, ctx, "ovfq_kv_append", side, args, (batch, rs)), q_out


def kv_append(cache, k, v, row_offsets, lengths, tables, q=None, q_out=None, rope=None, positions=None, max_rows=0, rows=None):
    """New tokens into the cache (ovfq_kv_append[_dev]): k and v [rows][kv_heads * head_dim], k turned by its position and both rounded to
    the cache's type; q [rows][heads * head_dim] turned likewise. k and v may be None together (queries only). positions
    [axes][rows] (int32): each token's place in its request if None. rows: of k, or of q alone as attend takes it. Returns the turned queries
    (None without q)."""
    call, q_out = _append_call(cache, k, v, row_offsets, lengths, tables, q, q_out, rope, positions, max_rows, rows)
    call()
    return q_out


def _attend_call(cache, q, row_offsets, lengths, tables, out, scale, window, max_rows, top, pages, rows=None, ctx=None):
    batch, side = _batch(row_offsets, lengths, tables, max_rows)
    qb = as_buf(q, np.float32, "q")
    rows = _query_rows(q, qb, rows, batch.requests, cache.head_dim)
    heads = qb.size // (rows * cache.head_dim)
    if heads % cache.kv_heads:
        raise OverfitArgumentError(f"heads ({heads}) must be a multiple of kv_heads ({cache.kv_heads})")
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise OverfitArgumentOutOfRangeError(f"scale ({scale}) must be finite")
    if window < 0:
        raise OverfitArgumentOutOfRangeError(f"window ({window}) must not be negative")
    if out is None:
        out = _empty(qb, qb.size).reshape(tuple(q.shape))
    yb = _sized(as_buf(out, np.float32, "out"), qb.size, "out")
    ob, lb, tb = side
    _apart("out", yb, q=qb, row_offsets=ob, lengths=lb, tables=tb)
    side += [qb, yb]
    args = (ctypes.byref(batch), qb.ptr, rows, heads, scale)
    if top is None:
        return _call(cache, ctx, "ovfq_attend", side, (*args, window, yb.ptr), batch), out
    if not 1 <= top <= _lib.MAX_TOP_PAGES:
        raise OverfitArgumentOutOfRangeError(f"top_pages ({top}) must be in [1, {_lib.MAX_TOP_PAGES}]")
    pb = _sized(as_buf(pages, np.int32, "pages", allow_none=True), rows * cache.kv_heads * top, "pages")
    _apart("pages", pb, q=qb, out=yb, row_offsets=ob, lengths=lb, tables=tb)
    side.append(pb)
    return _call(cache, ctx, "ovfq_attend_selected", side, (*args, top, yb.ptr, _ptr(pb)), batch), out


def attend(cache, q, row_offsets, lengths, tables, out=None, scale=None, window=0, max_rows=0, rows=None):
    """Attention of each request's new tokens, already appended, over its pages (ovfq_attend[_dev]): q [rows][heads * head_dim] or
    [rows][heads][head_dim] (laid out otherwise: `rows` says how many there are; without it a plane of one axis is one row), causal, over
    the last `window` tokens of each row (0: all). scale: 1 / sqrt(head_dim) if None. max_rows bounds every request's rows (0: not known),
    which sizes the launches: give 1 for a decode step. Returns the output, laid out as q."""
    call, out = _attend_call(cache, q, row_offsets, lengths, tables, out, scale, window, max_rows, None, None, rows)
    call()
    return out


def attend_selected(cache, q, row_offsets, lengths, tables, top_pages, out=None, pages=None, scale=None, max_rows=0, rows=None):
    """The same over top_pages pages for each row and key head (ovfq_attend_selected[_dev]): its own and the full pages before it whose mean
    key fits its queries best. The cache keeps sums. pages [rows][kv_heads][top_pages] (int32) receives them if given."""
    call, out = _attend_call(cache, q, row_offsets, lengths, tables, out, scale, 0, max_rows, top_pages, pages, rows)
    call()
    return out
