"""Outputs of the paged cache's operators that share memory with what the call reads (refused before any device work), and the entry points'
own checks on the device."""
import ctypes

import numpy as np
import pytest

import overfit_amd as ov
from overfit_amd import _lib
from test_kv_refusals import F, I, loose_cache

ROPE = dict(inv_freq=4, positions=3, pair_axes=4)  # sizes, beside the batch's


def batch(**change):
    return dict(dict(row_offsets=np.array([0, 1, 3], I), lengths=np.array([1, 40], I), tables=np.zeros((2, 2), I)), **change)


@pytest.mark.parametrize("name,size", [("row_offsets", 3), ("lengths", 2), ("tables", 4)])
@pytest.mark.parametrize("end", [0, 1])
def test_attention_over_the_batchs_arrays(name, size, end):
    mem = np.zeros(400, F)
    for plane in ("out", "pages"):
        n = 96 if plane == "out" else 12
        at = n - 1 if end else -size + 1
        call = batch(q=np.zeros((3, 32), F), out=np.zeros((3, 32), F), pages=np.zeros(12, I), top_pages=2)
        call[plane] = mem[100:100 + n] if plane == "out" else mem[100:100 + n].view(I)
        call[name] = mem[100 + at:100 + at + size].view(I).reshape(call[name].shape)
        cache = loose_cache()
        with pytest.raises(ov.OverfitArgumentError, match=f"{plane} overlaps {name}"):
            ov.attend_selected(cache, **call)
        if plane == "out":
            del call["pages"], call["top_pages"]
            with pytest.raises(ov.OverfitArgumentError, match=f"out overlaps {name}"):
                ov.attend(cache, **call)
        assert not cache.context.lib.calls


def test_pages_over_queries_and_outputs():
    mem = np.zeros(400, F)
    for other, at in (("q", 95), ("out", 95), ("q", -11), ("out", -11)):
        call = batch(q=np.zeros((3, 32), F), out=np.zeros((3, 32), F))
        call[other] = mem[100:196].reshape(3, 32)
        with pytest.raises(ov.OverfitArgumentError, match=f"pages overlaps {other}"):
            ov.attend_selected(loose_cache(), **call, top_pages=2, pages=mem[100 + at:112 + at].view(I))
    ov.attend_selected(loose_cache(), **call, top_pages=2, pages=mem[88:100].view(I))  # next to each other


@pytest.mark.parametrize("name,size", [("row_offsets", 3), ("lengths", 2), ("tables", 4), *ROPE.items()])
@pytest.mark.parametrize("end", [0, 1])
def test_turned_queries_over_inputs(name, size, end):
    mem = np.zeros(400, F)
    at = 47 if end else -size + 1
    shared = mem[100 + at:100 + at + size]
    arrays = dict(inv_freq=np.ones(4, F), pair_axes=np.zeros(4, I))
    call = batch(k=np.zeros(48, F), v=np.zeros(48, F), q=np.zeros((3, 16), F), q_out=mem[100:148].reshape(3, 16), positions=np.zeros(3, I))
    if name in arrays:
        arrays[name] = shared if name == "inv_freq" else shared.view(I)
    else:
        call[name] = shared.view(I).reshape(call[name].shape)
    cache = loose_cache()
    with pytest.raises(ov.OverfitArgumentError, match=f"q_out overlaps {name}"):
        ov.kv_append(cache, **call, rope=ov.Rope(arrays["inv_freq"], pair_axes=arrays["pair_axes"]))
    assert not cache.context.lib.calls


@pytest.mark.gpu
def test_entry_points():
    torch = pytest.importorskip("torch")
    cache = ov.KvCache(2, 16, 32, 4, sums=True)
    ctx, lib = cache.context, cache.context.lib
    x = torch.zeros(4000, device="cuda:0")
    ints = x.view(torch.int32)
    ints[1000:1002] = torch.tensor([0, 3], dtype=torch.int32)
    ints[1010], ints[1020] = 3, 0
    f = x.data_ptr()
    at = lambda n: f + 4 * n  # noqa: E731
    b = _lib.KvBatchStruct(1, 1, 0, at(1000), at(1010), at(1020))
    torch.cuda.synchronize()

    def selected(out, pages, q=0):
        return lib.ovfq_attend_selected_dev(ctx.handle, cache.handle, ctypes.byref(b), at(q), 3, 4, 1.0, 2, at(out), None if pages is None else at(pages))

    assert selected(200, None) == selected(200, 400) == selected(200, 392) == selected(200, 988) == _lib.OVFQ_OK
    for pages in (0, 191, 200, 391, 989, 1001, 1010, 1020, 1009):  # 12 of them, 192 queries and outputs
        assert selected(200, pages) == _lib.OVFQ_ERR_SIZE
    for out in (809, 1001, 1010, 1020):
        assert selected(out, None) == _lib.OVFQ_ERR_SIZE
        assert lib.ovfq_attend_dev(ctx.handle, cache.handle, ctypes.byref(b), f, 3, 4, 1.0, 0, at(out)) == _lib.OVFQ_ERR_SIZE

    def append(out):
        rope = _lib.RopeStruct(16, 0, 1, 1.0, at(2000), at(2010))
        return lib.ovfq_kv_append_dev(ctx.handle, cache.handle, ctypes.byref(b), at(3000), at(3100), 3, ctypes.byref(rope), at(2020), f, 4, at(out))

    assert append(0) == append(200) == append(2023) == _lib.OVFQ_OK
    for out in (809, 1001, 1010, 1020, 1809, 2007, 2010, 2017, 2020, 2022):
        assert append(out) == _lib.OVFQ_ERR_SIZE
    torch.cuda.synchronize()
