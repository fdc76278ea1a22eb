"""What a server runs around the shared quantized projections when one step holds rows of many requests: each request's
low-rank adapter beside a projection (AdapterSet, project_adapters), the norms around the residual sum (Norm,
residual_norm) and the verification of drafted tokens (verify_drafts).

As for the projections, numpy arrays use the synchronous host entry points and torch GPU tensors the ``_dev`` ones. The
Context.bind_*_dev methods convert a call's arguments once, for loops with buffers that stay.
"""
import ctypes
import math

import numpy as np

from . import _lib
from .errors import (OverfitArgumentError, OverfitArgumentNullError, OverfitArgumentOutOfRangeError,
                     OverfitUnsupportedTypeError, raise_for_status)
from .runtime import BoundCall, as_buf, default_context, same_side, torch

_ELEMENT = {_lib.TYPE_F32: "float32", _lib.TYPE_F16: "float16", _lib.TYPE_BF16: "bfloat16"}


def _as_elements(x, type_id, name, size):
    """(pointer, on the device, what holds the memory) of `size` contiguous elements of an adapter type."""
    if x is None:
        raise OverfitArgumentNullError(f"{name} is None")
    want = _ELEMENT[type_id]
    if torch is not None and isinstance(x, torch.Tensor):
        got, contiguous, n, where = str(x.dtype).split(".")[-1], x.is_contiguous(), x.numel(), (x.data_ptr(), x.is_cuda)
    elif isinstance(x, np.ndarray):
        got, contiguous, n, where = x.dtype.name, x.flags["C_CONTIGUOUS"], x.size, (x.ctypes.data, False)
    else:
        raise OverfitArgumentError(f"{name} must be a numpy array or a torch tensor")
    if got != want:
        raise OverfitArgumentError(f"{name} must have dtype {want}, got {got}")
    if not contiguous:
        raise OverfitArgumentError(f"{name} must be contiguous")
    if n != size:
        raise OverfitArgumentError(f"{name} has {n} elements, not {size}")
    return where + (x,)


class AdapterSet:
    """The low-rank adapters of one projection weight (ovfq_adapters_create): `slots` places, each empty or holding
    A [rank][input_size], B [output_size][rank] and a scale, rank <= max_rank, kept in `type_id` (TYPE_F32, TYPE_F16 or
    TYPE_BF16)."""

    def __init__(self, input_size: int, output_size: int, slots: int, max_rank: int, type_id=_lib.TYPE_F16, ctx=None):
        if type_id not in _ELEMENT:
            raise OverfitUnsupportedTypeError(f"adapter type {type_id}")
        if input_size <= 0 or output_size <= 0:
            raise OverfitArgumentOutOfRangeError(f"sizes ({input_size}, {output_size}) must be positive")
        if input_size % 32:
            raise OverfitArgumentError(f"input_size ({input_size}) must be a multiple of 32.")
        if not 1 <= slots <= _lib.MAX_ADAPTER_SLOTS:
            raise OverfitArgumentOutOfRangeError(f"slots ({slots}) must be in [1, {_lib.MAX_ADAPTER_SLOTS}]")
        if not 1 <= max_rank <= _lib.MAX_ADAPTER_RANK:
            raise OverfitArgumentOutOfRangeError(f"max_rank ({max_rank}) must be in [1, {_lib.MAX_ADAPTER_RANK}]")
        self._ctx = ctx or default_context()
        h = ctypes.c_void_p()
        raise_for_status(self._ctx.lib.ovfq_adapters_create(self._ctx.handle, type_id, input_size, output_size, slots,
                                                            max_rank, ctypes.byref(h)), self._ctx.lib)
        self.handle = h
        self.input_size, self.output_size, self.slots, self.max_rank = input_size, output_size, slots, max_rank
        self.type_id = type_id

    def __del__(self):
        h = getattr(self, "handle", None)
        if h is not None and h.value:
            try:
                self._ctx.lib.ovfq_adapters_destroy(h)
            except Exception:
                pass
            self.handle = None

    @property
    def context(self):
        return self._ctx

    @property
    def byte_count(self) -> int:
        n = ctypes.c_size_t()
        raise_for_status(self._ctx.lib.ovfq_adapters_info(self.handle, None, None, None, None, None, ctypes.byref(n)),
                         self._ctx.lib)
        return n.value

    def _check_slot(self, slot):
        if not 0 <= slot < self.slots:
            raise OverfitArgumentOutOfRangeError(f"slot {slot} out of range [0, {self.slots})")

    def load(self, slot: int, a, b, scale: float = 1.0):
        """Puts a [rank][input_size] and b [output_size][rank] (numpy arrays or torch tensors of the set's type, both on
        the host or both on the device) into `slot`; scale is usually alpha / rank."""
        self._check_slot(slot)
        if a is None or b is None:
            raise OverfitArgumentNullError("a / b is None")
        if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[0] != b.shape[1]:
            raise OverfitArgumentError("a must be [rank][input_size] and b [output_size][rank]")
        rank = int(a.shape[0])
        if not 1 <= rank <= self.max_rank:
            raise OverfitArgumentOutOfRangeError(f"rank ({rank}) must be in [1, {self.max_rank}]")
        if a.shape[1] != self.input_size or b.shape[0] != self.output_size:
            raise OverfitArgumentError(f"a must have {self.input_size} columns and b {self.output_size} rows")
        pa, da, _ka = _as_elements(a, self.type_id, "a", rank * self.input_size)
        pb, db, _kb = _as_elements(b, self.type_id, "b", rank * self.output_size)
        if da != db:
            raise OverfitArgumentError("host and device buffers cannot be mixed in one call")
        if da and {a.device.index, b.device.index} != {self._ctx.device}:
            raise OverfitArgumentError("a, b and the set must be on one device")
        fn = self._ctx.lib.ovfq_adapters_load_dev if da else self._ctx.lib.ovfq_adapters_load
        raise_for_status(fn(self.handle, slot, pa, pb, rank, float(scale)), self._ctx.lib)

    def unload(self, slot: int):
        """Empties `slot`: rows that name it get the projection alone."""
        self._check_slot(slot)
        raise_for_status(self._ctx.lib.ovfq_adapters_unload(self.handle, slot), self._ctx.lib)


def _empty(like, n, dtype=np.float32):
    """An uninitialised output beside `like`: a device tensor for a device buffer, else a numpy array."""
    if like.device:
        return torch.empty(n, dtype={np.float32: torch.float32, np.int32: torch.int32}[dtype], device=like.obj.device)
    return np.zeros(n, dtype)


def _context(ctx, bufs):
    """The context that a call on these buffers runs on: the given one, or the default one of the tensors' device."""
    devices = {b.obj.device.index for b in bufs if b is not None and b.device}
    if len(devices) > 1 or (ctx is not None and devices - {ctx.device}):
        raise OverfitArgumentError("the call's tensors and its context must be on one device")
    return ctx or default_context(*devices)


def _sized(b, n, name):
    if b is not None and b.size < n:
        raise OverfitArgumentError(f"{name} has {b.size} elements, {n} are needed")
    return b


def _ptr(b):
    return None if b is None else b.ptr


def _adapters_call(weights, adapters, x, row_slots, rows, biases, outs, ctx=None):
    n = len(weights)
    if not 1 <= n <= 4:
        raise OverfitArgumentOutOfRangeError(f"{n} weights: 1 to 4 are taken")
    if len(adapters) != n or (outs is not None and len(outs) != n) or (biases is not None and len(biases) != n):
        raise OverfitArgumentError("weights, adapters, outs and biases must have the same length")
    if rows <= 0:
        raise OverfitArgumentOutOfRangeError(f"rows ({rows}) must be positive")
    xb = _sized(as_buf(x, np.float32, "x"), rows * weights[0].InputSize, "x")
    sb = _sized(as_buf(row_slots, np.int32, "row_slots"), rows, "row_slots")
    if outs is None:
        outs = [_empty(xb, rows * w.OutputSize) for w in weights]
    ob = [_sized(as_buf(o, np.float32, "out"), rows * w.OutputSize, "out") for o, w in zip(outs, weights)]
    bb = [as_buf(b, np.float32, "bias", allow_none=True) for b in (biases or [None] * n)]
    bb = [None if b is None or b.size == 0 else _sized(b, w.OutputSize, "bias") for b, w in zip(bb, weights)]
    dev = same_side(xb, sb, *ob, *bb)
    if ctx is not None and ctx is not weights[0].context:
        raise OverfitArgumentError("the weights belong to another context")
    ctx = _context(weights[0].context, [xb, sb, *ob, *bb])
    arr = ctypes.c_void_p * n
    args = (ctx.handle, n, arr(*[w.handle.value for w in weights]),
            arr(*[None if s is None else s.handle.value for s in adapters]), xb.ptr, rows, sb.ptr,
            arr(*[_ptr(b) for b in bb]), arr(*[o.ptr for o in ob]))
    fn = ctx.lib.ovfq_project_adapters_dev if dev else ctx.lib.ovfq_project_adapters
    return BoundCall(ctx, fn, args, (list(weights), list(adapters), [xb, sb, *ob, *bb])), outs


def project_adapters(weights, adapters, x, row_slots, rows=1, biases=None, outs=None):
    """project_multi with each row's adapter added (ovfq_project_adapters[_dev]): outs[i][m] = (biases[i] +)
    W_i q(x[m]) + scale_s B_s (A_s x[m]), s = row_slots[m] (int32) of adapters[i] (an AdapterSet, or None). A row whose slot
    is negative, past the set or empty gets the projection alone. Returns the outputs."""
    call, outs = _adapters_call(weights, adapters, x, row_slots, rows, biases, outs)
    call()
    return outs


class Norm:
    """A norm over the channels: kind "rms" or "layer", weight and bias [k] (None: ones, none) and eps."""

    __slots__ = ("weight", "bias", "eps", "kind")
    KINDS = {"rms": 0, "layer": 1}

    def __init__(self, weight=None, bias=None, eps=1e-5, kind="rms"):
        if kind not in self.KINDS:
            raise OverfitArgumentError(f"norm kind must be one of {sorted(self.KINDS)}, not {kind!r}")
        if not (math.isfinite(eps) and eps >= 0):
            raise OverfitArgumentOutOfRangeError(f"eps ({eps}) must be finite and not negative")
        self.weight, self.bias, self.eps, self.kind = weight, bias, float(eps), kind


GATE_AXES = {None: 0, "channel": 1, "row": 2, "full": 3}


def _norm_call(y, rows, residual, post, gate, gate_axis, scale, pre, h_out, x_out, ctx, need_h):
    yb = as_buf(y, np.float32, "y")
    if rows <= 0:
        raise OverfitArgumentOutOfRangeError(f"rows ({rows}) must be positive")
    if yb.size == 0 or yb.size % rows:
        raise OverfitArgumentError(f"y has {yb.size} elements, not a whole number for each of {rows} rows")
    k = yb.size // rows
    if gate_axis not in GATE_AXES:
        raise OverfitArgumentError(f"gate_axis must be 'channel', 'row' or 'full', not {gate_axis!r}")
    if (gate is None) != (gate_axis is None):
        raise OverfitArgumentError("gate and gate_axis go together")
    if pre is None and x_out is not None:
        raise OverfitArgumentError("x_out without a pre norm")
    if h_out is None and (need_h or pre is None):
        h_out = _empty(yb, rows * k)
    if x_out is None and pre is not None:
        x_out = _empty(yb, rows * k)
    rb = _sized(as_buf(residual, np.float32, "residual", allow_none=True), rows * k, "residual")
    gb = _sized(as_buf(gate, np.float32, "gate", allow_none=True),
                {None: 0, "channel": k, "row": rows, "full": rows * k}[gate_axis], "gate")
    hb = _sized(as_buf(h_out, np.float32, "h_out", allow_none=True), rows * k, "h_out")
    xb = _sized(as_buf(x_out, np.float32, "x_out", allow_none=True), rows * k, "x_out")
    side = [yb, rb, gb, hb, xb]
    norms = []
    for name, n in (("post", post), ("pre", pre)):
        if n is None:
            norms.append(None)
            continue
        if not isinstance(n, Norm):
            raise OverfitArgumentError(f"{name} must be a Norm")
        w = _sized(as_buf(n.weight, np.float32, f"{name} weight", allow_none=True), k, f"{name} weight")
        b = _sized(as_buf(n.bias, np.float32, f"{name} bias", allow_none=True), k, f"{name} bias")
        side += [w, b]
        norms.append(_lib.NormStruct(Norm.KINDS[n.kind], n.eps, _ptr(w), _ptr(b)))
    dev = same_side(*side)
    ctx = _context(ctx, side)
    fn = ctx.lib.ovfq_residual_norm_dev if dev else ctx.lib.ovfq_residual_norm
    args = (ctx.handle, yb.ptr, _ptr(rb), rows, k, None if norms[0] is None else ctypes.byref(norms[0]), _ptr(gb),
            GATE_AXES[gate_axis], float(scale), None if norms[1] is None else ctypes.byref(norms[1]), _ptr(hb), _ptr(xb))
    return BoundCall(ctx, fn, args, (side, norms)), h_out, x_out


def residual_norm(y, rows, residual=None, post=None, gate=None, gate_axis=None, scale=1.0, pre=None, h_out=None,
                  x_out=None, ctx=None):
    """The step between two blocks (ovfq_residual_norm[_dev]) over `rows` rows: h = residual + scale * gate * post(y),
    x = pre(h), with post and pre each a Norm or None, and gate [k], [rows] or [rows][k] by gate_axis "channel", "row" or
    "full". Returns (h, x); x is None without a pre norm, and h is not computed into memory (None) for a plain norm: no
    residual, post, gate or h_out, and a pre norm."""
    need_h = residual is not None or post is not None or gate is not None
    call, h_out, x_out = _norm_call(y, rows, residual, post, gate, gate_axis, scale, pre, h_out, x_out, ctx, need_h)
    call()
    return h_out, x_out


def _verify_call(logits, vocab, row_offsets, draft_tokens, accept_uniforms, final_uniforms, draft_probs, temperature,
                 accepted, tokens, ctx):
    if vocab <= 0:
        raise OverfitArgumentOutOfRangeError(f"vocab ({vocab}) must be positive")
    lb = as_buf(logits, np.float32, "logits")
    if lb.size == 0 or lb.size % vocab:
        raise OverfitArgumentError(f"logits has {lb.size} elements, not whole rows of {vocab}")
    rows = lb.size // vocab
    rb = as_buf(row_offsets, np.int32, "row_offsets")
    requests = rb.size - 1
    if requests < 1:
        raise OverfitArgumentError("row_offsets needs an entry for each request and one more")
    if requests > rows:
        raise OverfitArgumentError(f"{requests} requests need as many rows of logits at least, got {rows}")
    drafts = rows - requests
    none = lambda v: None if drafts == 0 else v  # noqa: E731
    tb = _sized(as_buf(draft_tokens, np.int32, "draft_tokens", allow_none=not drafts), drafts, "draft_tokens")
    ub = _sized(as_buf(accept_uniforms, np.float32, "accept_uniforms", allow_none=not drafts), drafts, "accept_uniforms")
    fb = _sized(as_buf(final_uniforms, np.float32, "final_uniforms"), requests, "final_uniforms")
    qb = _sized(as_buf(draft_probs, np.float32, "draft_probs", allow_none=True), drafts * vocab, "draft_probs")
    pb = _sized(as_buf(temperature, np.float32, "temperature", allow_none=True), requests, "temperature")
    accepted = _empty(lb, requests, np.int32) if accepted is None else accepted
    tokens = _empty(lb, rows, np.int32) if tokens is None else tokens
    ab = _sized(as_buf(accepted, np.int32, "accepted"), requests, "accepted")
    ob = _sized(as_buf(tokens, np.int32, "tokens"), rows, "tokens")
    side = [lb, rb, none(tb), none(ub), fb, none(qb), pb, ab, ob]
    dev = same_side(*side)
    ctx = _context(ctx, side)
    fn = ctx.lib.ovfq_verify_drafts_dev if dev else ctx.lib.ovfq_verify_drafts
    args = (ctx.handle, lb.ptr, rows, vocab, requests, rb.ptr, _ptr(none(tb)), _ptr(none(qb)), _ptr(pb), _ptr(none(ub)),
            fb.ptr, ab.ptr, ob.ptr)
    return BoundCall(ctx, fn, args, side), accepted, tokens


def verify_drafts(logits, vocab, row_offsets, draft_tokens, accept_uniforms, final_uniforms, draft_probs=None,
                  temperature=None, accepted=None, tokens=None, ctx=None):
    """Speculative decoding's check of drafted tokens against the LM head's logits [rows][vocab] (ovfq_verify_drafts[_dev],
    which says how rows, drafts and random numbers are laid out). Returns (accepted [requests], tokens [rows])."""
    call, accepted, tokens = _verify_call(logits, vocab, row_offsets, draft_tokens, accept_uniforms, final_uniforms,
                                          draft_probs, temperature, accepted, tokens, ctx)
    call()
    return accepted, tokens
