"""Arguments that the paged cache's operators refuse before any device work (no GPU needed)."""
import ctypes

import numpy as np
import pytest

import overfit_amd as ov
from overfit_amd import _lib

F = np.float32
I = np.int32  # noqa: E741


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def fn(*args):
            self.calls.append(name)
            return 0

        fn.__name__ = name
        return fn


def loose_cache(kv_heads=2, head_dim=8, page_size=32, pages=4, sums=True):
    """A cache without a device: what the calls check before they call the library."""
    ctx = ov.Context.__new__(ov.Context)
    ctx.lib, ctx.handle, ctx.device = Library(), ctypes.c_void_p(16), 0
    c = ov.KvCache.__new__(ov.KvCache)
    c.kv_heads, c.head_dim, c.page_size, c.pages, c.sums, c.type_id = kv_heads, head_dim, page_size, pages, sums, ov.TYPE_F16
    c._ctx, c.handle = ctx, ctypes.c_void_p(0)
    return c


@pytest.mark.parametrize("args,error", [
    ((0, 64, 64, 4), ov.OverfitArgumentOutOfRangeError),
    ((1025, 64, 64, 4), ov.OverfitArgumentOutOfRangeError),
    ((2, 0, 64, 4), ov.OverfitArgumentOutOfRangeError),
    ((2, 264, 64, 4), ov.OverfitArgumentOutOfRangeError),
    ((2, 60, 64, 4), ov.OverfitArgumentError),
    ((2, 64, 16, 4), ov.OverfitArgumentOutOfRangeError),
    ((2, 64, 48, 4), ov.OverfitArgumentOutOfRangeError),
    ((2, 64, 512, 4), ov.OverfitArgumentOutOfRangeError),
    ((2, 64, 64, 0), ov.OverfitArgumentOutOfRangeError),
    ((2, 64, 256, 1 << 23), ov.OverfitArgumentError),
    ((2, 64, 64, 4, ov.TYPE_F32), ov.OverfitUnsupportedTypeError),
    ((2, 64, 64, 4, ov.TYPE_Q8_0), ov.OverfitUnsupportedTypeError),
])
def test_cache_sizes(args, error):
    with pytest.raises(error):
        ov.KvCache(*args)


def test_rope_arguments():
    with pytest.raises(ov.OverfitArgumentError):
        ov.Rope(np.ones(4, F), "quarters")
    with pytest.raises(ov.OverfitArgumentOutOfRangeError):
        ov.Rope(np.ones(4, F), scale=float("inf"))
    with pytest.raises(ov.OverfitArgumentNullError):
        ov.Rope(None)


BATCH = dict(row_offsets=np.array([0, 1, 3], I), lengths=np.array([1, 40], I), tables=np.zeros((2, 2), I))


@pytest.mark.parametrize("change,error", [
    (dict(row_offsets=None), ov.OverfitArgumentNullError),
    (dict(row_offsets=np.zeros(1, I)), ov.OverfitArgumentError),
    (dict(row_offsets=np.zeros(3, np.int64)), ov.OverfitArgumentError),
    (dict(lengths=np.zeros(1, I)), ov.OverfitArgumentError),
    (dict(tables=np.zeros(3, I)), ov.OverfitArgumentError),
    (dict(tables=np.zeros(0, I)), ov.OverfitArgumentError),
    (dict(tables=np.zeros((3, 2), I).T), ov.OverfitArgumentError),  # not contiguous
    (dict(max_rows=-1), ov.OverfitArgumentOutOfRangeError),
    (dict(k=None), ov.OverfitArgumentNullError),
    (dict(k=None, v=None), ov.OverfitArgumentNullError),
    (dict(k=np.zeros(47, F)), ov.OverfitArgumentError),
    (dict(k=np.zeros(32, F)), ov.OverfitArgumentError),  # not as many as v
    (dict(k=np.zeros(48, np.float64)), ov.OverfitArgumentError),
    (dict(q=np.zeros((3, 32), F)), ov.OverfitArgumentNullError),  # no rope
    (dict(q=np.zeros((3, 24), F), rope=ov.Rope(np.ones(4, F))), ov.OverfitArgumentError),  # 3 heads over 2
    (dict(q=np.zeros(50, F), rope=ov.Rope(np.ones(4, F))), ov.OverfitArgumentError),
    (dict(q=np.zeros((3, 32), F), q_out=np.zeros(95, F), rope=ov.Rope(np.ones(4, F))), ov.OverfitArgumentError),
    (dict(q_out=np.zeros(96, F)), ov.OverfitArgumentNullError),
    (dict(rope="pairs"), ov.OverfitArgumentError),
    (dict(rope=ov.Rope(np.ones(5, F))), ov.OverfitArgumentOutOfRangeError),
    (dict(rope=ov.Rope(np.ones(0, F))), ov.OverfitArgumentOutOfRangeError),
    (dict(rope=ov.Rope(np.ones(4, F), pair_axes=np.zeros(3, I))), ov.OverfitArgumentError),
    (dict(positions=np.zeros(3, I)), ov.OverfitArgumentNullError),  # no rope
    (dict(rope=ov.Rope(np.ones(4, F)), positions=np.zeros(4, I)), ov.OverfitArgumentError),
    (dict(rope=ov.Rope(np.ones(4, F)), positions=np.zeros(15, I)), ov.OverfitArgumentOutOfRangeError),  # five axes
])
def test_append_arguments(change, error):
    cache = loose_cache()
    call = dict(BATCH, k=np.zeros(48, F), v=np.zeros(48, F))
    call.update(change)
    with pytest.raises(error):
        ov.kv_append(cache, **call)
    assert not cache.context.lib.calls


@pytest.mark.parametrize("selected", [False, True])
@pytest.mark.parametrize("change,error", [
    (dict(row_offsets=np.zeros(1, I)), ov.OverfitArgumentError),
    (dict(lengths=None), ov.OverfitArgumentNullError),
    (dict(q=None), ov.OverfitArgumentNullError),
    (dict(q=np.zeros((0, 32), F)), ov.OverfitArgumentError),
    (dict(q=np.zeros((3, 24), F)), ov.OverfitArgumentError),
    (dict(q=np.zeros((3, 30), F)), ov.OverfitArgumentError),
    (dict(out=np.zeros(95, F)), ov.OverfitArgumentError),
    (dict(scale=float("nan")), ov.OverfitArgumentOutOfRangeError),
    (dict(max_rows=-1), ov.OverfitArgumentOutOfRangeError),
])
def test_attend_arguments(selected, change, error):
    cache = loose_cache()
    call = dict(BATCH, q=np.zeros((3, 32), F))
    call.update(change)
    with pytest.raises(error):
        ov.attend_selected(cache, top_pages=2, **call) if selected else ov.attend(cache, **call)
    assert not cache.context.lib.calls


@pytest.mark.parametrize("fn,change,error", [
    ("attend", dict(window=-1), ov.OverfitArgumentOutOfRangeError),
    ("attend_selected", dict(top_pages=0), ov.OverfitArgumentOutOfRangeError),
    ("attend_selected", dict(top_pages=4097), ov.OverfitArgumentOutOfRangeError),
    ("attend_selected", dict(top_pages=2, pages=np.zeros(11, I)), ov.OverfitArgumentError),
])
def test_other_attend_arguments(fn, change, error):
    with pytest.raises(error):
        getattr(ov, fn)(loose_cache(), np.zeros((3, 32), F), **BATCH, **change)


def test_outputs_that_are_inputs():
    q = np.zeros((3, 32), F)
    with pytest.raises(ov.OverfitArgumentError):
        ov.attend(loose_cache(), q, **BATCH, out=q)
    k = np.zeros(48, F)
    with pytest.raises(ov.OverfitArgumentError):
        ov.kv_append(loose_cache(), k, np.zeros(48, F), **BATCH, q=np.zeros((3, 16), F), q_out=k, rope=ov.Rope(np.ones(4, F)))


def test_prepared_calls_need_outputs_and_device_tensors():
    cache = loose_cache()
    q = np.zeros((3, 32), F)
    with pytest.raises(ValueError):
        cache.context.bind_attend_dev(cache, q, **BATCH, out=None)
    with pytest.raises(ValueError):
        cache.context.bind_attend_selected_dev(cache, q, **BATCH, top_pages=2, out=None)
    with pytest.raises(ValueError):
        cache.context.bind_kv_append_dev(cache, None, None, **BATCH, q=q, rope=ov.Rope(np.ones(4, F)))
    with pytest.raises(ov.OverfitArgumentError):
        cache.context.bind_attend_dev(cache, q, **BATCH, out=np.zeros(96, F))
    with pytest.raises(ov.OverfitArgumentError):
        loose_cache().context.bind_attend_dev(cache, q, **BATCH, out=np.zeros(96, F))  # another context


def test_entry_points_refuse_null():
    lib = _lib.load()
    h = ctypes.c_void_p()
    b = _lib.KvBatchStruct()
    assert lib.ovfq_kv_create(None, 1, 1, 64, 64, 1, 0, ctypes.byref(h)) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_kv_destroy(None) == _lib.OVFQ_ERR_NULL
    assert lib.ovfq_kv_info(None, *[None] * 9) == _lib.OVFQ_ERR_NULL
    for fn in (lib.ovfq_kv_append, lib.ovfq_kv_append_dev):
        assert fn(None, None, ctypes.byref(b), None, None, 1, None, None, None, 0, None) == _lib.OVFQ_ERR_NULL
    for fn in (lib.ovfq_attend, lib.ovfq_attend_dev):
        assert fn(None, None, ctypes.byref(b), None, 1, 1, 1.0, 0, None) == _lib.OVFQ_ERR_NULL
    for fn in (lib.ovfq_attend_selected, lib.ovfq_attend_selected_dev):
        assert fn(None, None, ctypes.byref(b), None, 1, 1, 1.0, 4, None, None) == _lib.OVFQ_ERR_NULL


@pytest.mark.parametrize("at", [0, 1, 95])
def test_outputs_that_overlap_inputs(at):
    mem = np.zeros(400, F)
    with pytest.raises(ov.OverfitArgumentError):
        ov.attend(loose_cache(), mem[:96].reshape(3, 32), **BATCH, out=mem[at:at + 96].reshape(3, 32))
    call = dict(BATCH, k=mem[:48], v=np.zeros(48, F), q=np.zeros((3, 16), F), rope=ov.Rope(np.ones(4, F)))
    with pytest.raises(ov.OverfitArgumentError):
        ov.kv_append(loose_cache(), **call, q_out=mem[at // 2:at // 2 + 48].reshape(3, 16))
    call["k"], call["v"] = call["v"], call["k"]
    with pytest.raises(ov.OverfitArgumentError):
        ov.kv_append(loose_cache(), **call, q_out=mem[at // 2:at // 2 + 48].reshape(3, 16))
    if at:
        call.update(v=np.zeros(48, F), q=mem[:48].reshape(3, 16))
        with pytest.raises(ov.OverfitArgumentError):
            ov.kv_append(loose_cache(), **call, q_out=mem[at // 4 + 1:at // 4 + 49].reshape(3, 16))
