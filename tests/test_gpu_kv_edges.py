"""Edges of the paged cache's operators on the device: what they refuse, lifetime, capture, planes at any four bytes, more requests than a
wave has lanes, caches past 4 GiB, several threads, contexts and streams."""
import ctypes
import gc
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, Requests, as_stored, attention, case, check  # noqa: E402
from overfit_amd import _lib  # noqa: E402
from test_gpu_attend_selected import choose  # noqa: E402

I = np.int32  # noqa: E741


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_a_context_outlives_its_caches():
    ctx = ov.Context(0)
    cache = ov.KvCache(1, 64, 32, 2, ctx=ctx)
    assert ctx.lib.ovfq_ctx_destroy(ctx.handle) == _lib.OVFQ_ERR_STATE and b"cache" in ctx.lib.ovfq_last_error()
    view = cache.key_view()
    del cache
    gc.collect()
    assert ctx.lib.ovfq_ctx_destroy(ctx.handle) == _lib.OVFQ_ERR_STATE  # the view holds it
    assert not view.float().any()
    del view
    gc.collect()
    ctx.close()


def test_caches_of_other_contexts_are_refused():
    ctx = ov.Context(0)
    cache = ov.KvCache(1, 64, 32, 2)
    x = torch.zeros(1, 64, device=DEV)
    with pytest.raises(ov.OverfitArgumentError):
        ctx.bind_attend_dev(cache, x, i32([0, 1]), i32([1]), i32([[0]]), torch.zeros_like(x))
    b = _lib.KvBatchStruct(1, 1, 0, 16, 16, 16)
    rc = ctx.lib.ovfq_attend_dev(ctx.handle, cache.handle, ctypes.byref(b), x.data_ptr(), 1, 1, 1.0, 0, x.data_ptr())
    assert rc == _lib.OVFQ_ERR_SIZE
    ctx.close()


@pytest.mark.parametrize("change,error", [
    (dict(row_offsets=[1, 3]), ov.OverfitArgumentError),
    (dict(row_offsets=[0, 2]), ov.OverfitArgumentError),
    (dict(row_offsets=[0, 4]), ov.OverfitArgumentError),
    (dict(row_offsets=[0, 2, 1, 3], lengths=[3] * 3, tables=[[0, 1]] * 3), ov.OverfitArgumentError),
    (dict(lengths=[2]), ov.OverfitArgumentError),
    (dict(lengths=[65]), ov.OverfitArgumentError),
    (dict(lengths=[33], tables=[[0, 4]]), ov.OverfitArgumentOutOfRangeError),
    (dict(lengths=[33], tables=[[0, -1]]), ov.OverfitArgumentOutOfRangeError),
    (dict(max_rows=2), ov.OverfitArgumentError),
])
def test_host_arrays_that_do_not_fit(change, error):
    cache = ov.KvCache(1, 8, 32, 4, sums=True)
    call = dict(row_offsets=[0, 3], lengths=[3], tables=[[0, 1]], max_rows=0)
    call.update(change)
    most = call.pop("max_rows")
    b = [np.array(call[k], I) for k in ("row_offsets", "lengths", "tables")]
    x = np.zeros((3, 8), np.float32)
    for fn in (lambda: ov.kv_append(cache, x, x, *b, max_rows=most), lambda: ov.attend(cache, x, *b, max_rows=most),
               lambda: ov.attend_selected(cache, x, *b, 2, max_rows=most)):
        with pytest.raises(error):
            fn()


def test_host_arrays_with_pages_in_common():
    """Requests that share pages may read them, not write them; pages before a window may be gone."""
    cache = ov.KvCache(1, 8, 32, 4)
    x = np.zeros((2, 8), np.float32)
    off, tables = np.array([0, 1, 2], I), np.array([[0, 1], [0, 2]], I)
    with pytest.raises(ov.OverfitArgumentError):
        ov.kv_append(cache, x, x, off, np.array([32, 5], I), tables)
    ov.kv_append(cache, x, x, off, np.array([33, 40], I), tables)
    ov.attend(cache, x, off, np.array([32, 5], I), tables)
    gone = np.array([[-1, 1], [-1, 2]], I)
    with pytest.raises(ov.OverfitArgumentOutOfRangeError):
        ov.attend(cache, x, off, np.array([33, 40], I), gone, window=2)
    ov.attend(cache, x, off, np.array([34, 40], I), gone, window=2)


def test_other_refusals():
    cache = ov.KvCache(1, 64, 32, 2)
    lib, ctx = cache.context.lib, cache.context
    x = torch.zeros(1, 64, device=DEV)
    with pytest.raises(ov.OverfitInvalidOperationError):  # no sums
        ov.attend_selected(cache, x, i32([0, 1]), i32([1]), i32([[0]]), 2)
    with pytest.raises(ov.OverfitArgumentError):
        cache.sum_view()
    with pytest.raises(ov.OverfitUnsupportedTypeError):
        cache.scale_view()
    off, length, table = i32([0, 1]), i32([1]), i32([[0]])
    b = _lib.KvBatchStruct(1, 1, 0, off.data_ptr(), length.data_ptr(), table.data_ptr())
    p = x.data_ptr()

    def attend(batch=b, q=p, rows=1, heads=1, scale=1.0, window=0, out=p):
        return lib.ovfq_attend_dev(ctx.handle, cache.handle, None if batch is None else ctypes.byref(batch), q, rows, heads, scale, window, out)

    change = lambda **k: attend(batch=_lib.KvBatchStruct(*[k.get(n, getattr(b, n)) for n, _ in b._fields_]))  # noqa: E731
    assert attend(batch=None) == _lib.OVFQ_ERR_NULL and attend(q=None) == _lib.OVFQ_ERR_NULL and attend(out=None) == _lib.OVFQ_ERR_NULL
    assert attend(rows=0) == _lib.OVFQ_ERR_RANGE and attend(rows=65537) == _lib.OVFQ_ERR_RANGE
    assert attend(heads=0) == _lib.OVFQ_ERR_RANGE and attend(scale=float("inf")) == _lib.OVFQ_ERR_RANGE
    assert attend(window=-1) == _lib.OVFQ_ERR_RANGE and attend(q=p + 2) == _lib.OVFQ_ERR_SIZE
    assert change(requests=0) == _lib.OVFQ_ERR_RANGE and change(requests=65537) == _lib.OVFQ_ERR_RANGE
    assert change(table_width=0) == _lib.OVFQ_ERR_RANGE and change(max_rows=-1) == _lib.OVFQ_ERR_RANGE
    assert change(requests=65536, table_width=65536) == _lib.OVFQ_ERR_SIZE
    assert change(lengths=None) == _lib.OVFQ_ERR_NULL and change(lengths=length.data_ptr() + 2) == _lib.OVFQ_ERR_SIZE
    assert attend(rows=65536, heads=1024) == _lib.OVFQ_ERR_SIZE  # 2^32 values
    many = ov.KvCache(128, 8, 32, 1)
    assert lib.ovfq_attend_dev(ctx.handle, many.handle, ctypes.byref(b), p, 65536, 128, 1.0, 0, p) == _lib.OVFQ_ERR_SIZE
    wide = ov.KvCache(1, 256, 32, 1, sums=True)
    assert lib.ovfq_attend_selected_dev(ctx.handle, wide.handle, ctypes.byref(b), p, 1, 65, 1.0, 2, p, None) == _lib.OVFQ_ERR_SIZE
    assert lib.ovfq_attend_selected_dev(ctx.handle, wide.handle, ctypes.byref(b), p, 1, 1, 1.0, 0, p, None) == _lib.OVFQ_ERR_RANGE

    def append(k=p, v=p, rope=None, positions=None, q=None, heads=0, q_out=None):
        return lib.ovfq_kv_append_dev(ctx.handle, cache.handle, ctypes.byref(b), k, v, 1, None if rope is None else ctypes.byref(rope), positions, q,
                                      heads, q_out)

    rope = lambda *v: _lib.RopeStruct(*v)  # noqa: E731
    assert append(v=None) == _lib.OVFQ_ERR_NULL and append(k=None, v=None) == _lib.OVFQ_ERR_NULL
    assert append(q=p, heads=1, q_out=p) == _lib.OVFQ_ERR_NULL and append(positions=p) == _lib.OVFQ_ERR_NULL
    assert append(rope=rope(64, 0, 1, 1.0, p, None), q=p, heads=1) == _lib.OVFQ_ERR_NULL
    for bad, rc in ((rope(0, 0, 1, 1.0, p, None), _lib.OVFQ_ERR_RANGE), (rope(66, 0, 1, 1.0, p, None), _lib.OVFQ_ERR_RANGE),
                    (rope(7, 0, 1, 1.0, p, None), _lib.OVFQ_ERR_SIZE), (rope(64, 2, 1, 1.0, p, None), _lib.OVFQ_ERR_RANGE),
                    (rope(64, 0, 0, 1.0, p, None), _lib.OVFQ_ERR_RANGE), (rope(64, 0, 5, 1.0, p, None), _lib.OVFQ_ERR_RANGE),
                    (rope(64, 0, 1, float("nan"), p, None), _lib.OVFQ_ERR_RANGE), (rope(64, 0, 1, 1.0, None, None), _lib.OVFQ_ERR_NULL),
                    (rope(64, 0, 1, 1.0, p, p + 1), _lib.OVFQ_ERR_SIZE)):
        assert append(rope=bad) == rc
    with pytest.raises(ov.OverfitArgumentOutOfRangeError):  # an axis that there is none of, checked on the host
        ov.kv_append(cache, np.zeros(64, np.float32), np.zeros(64, np.float32), np.array([0, 1], I), np.array([1], I), np.zeros((1, 1), I),
                     rope=ov.Rope(np.ones(2, np.float32), pair_axes=np.array([0, 4], I)))


def test_no_cache_is_made_while_a_stream_is_captured():
    stream, ctx = torch.cuda.Stream(), ov.Context(0)
    ctx.set_stream(stream.cuda_stream)
    cache = ov.KvCache(1, 64, 32, 2, ctx=ctx)
    x, out = torch.ones(1, 64, device=DEV), torch.zeros(1, 64, device=DEV)
    b = (i32([0, 1]), i32([1]), i32([[1]]))
    with torch.cuda.stream(stream):
        ov.kv_append(cache, x, x, *b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    call = ctx.bind_attend_dev(cache, x, *b, out)
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(ov.OverfitInvalidOperationError):
            ov.KvCache(1, 64, 32, 2, ctx=ctx)
        call()  # the context's first call: it grows its scratch meanwhile
    del call
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert (out == 1).all()
    # destroyed while captured: the memory stays until the context gives it back
    before = ctx.scratch_bytes()[1]
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other, stream=stream):
        out.zero_()
        n = cache.byte_count
        del cache
        gc.collect()
    assert ctx.scratch_bytes()[1] == before + n
    del graph
    ctx.release_retired()
    assert ctx.scratch_bytes()[1] == 0
    ctx.close()


def test_graphs_that_share_a_workspace():
    """Two graphs of one context, of different sizes, replayed in turn, on the default stream's context as well."""
    rng = np.random.default_rng(1)
    ctx, stream = ov.default_context(), torch.cuda.Stream()
    reqs = [Requests(ov, rng, "f16", 2, 64, 32, c, m, sums=True).fill() for c, m in (((1, 1), (3000, 70)), ((40,), (2000,)))]
    qs = [rng.standard_normal((r.rows, 256)).astype(np.float32) for r in reqs]
    outs = [torch.empty(r.rows, 256, device=DEV) for r in reqs]
    calls = [ctx.bind_attend_dev(r.cache, r.t(q), *r.batch(), o) for r, q, o in zip(reqs, qs, outs)]
    few = [torch.empty(r.rows, 256, device=DEV) for r in reqs]
    calls += [ctx.bind_attend_selected_dev(r.cache, r.t(q), *r.batch(), 9, o) for r, q, o in zip(reqs, qs, few)]
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graphs = []
        for call in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                call()
            graphs.append(g)
        want = [attention(r, q, 4) for r, q in zip(reqs, qs)]
        for r, q in zip(reqs, qs):
            pages = choose(r, q, 4, 9)
            want.append(attention(r, q, 4, keep=lambda row, a, seen: np.isin(seen // 32, pages[row, a])))
        for _ in range(3):
            for o in outs + few:
                o.fill_(7)
            torch.cuda.synchronize()
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            for o, (w, e) in zip(outs + few, want):
                check(o, w, e)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


def odd(x):
    """The same values at an address that is a multiple of four bytes only."""
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)
    flat[1:].copy_(x.reshape(-1))
    return flat[1:].view(x.shape)


@pytest.mark.parametrize("type_", ["f16", "i8"])
@pytest.mark.parametrize("style", ["pairs", "halves"])
def test_planes_at_any_four_bytes(type_, style):
    made = []
    for shift in (lambda x: x, odd):
        req = Requests(ov, np.random.default_rng(3), type_, 2, 64, 32, [3, 40], [0, 0], sums=True)
        k, v = (shift(req.t(np.concatenate(x).reshape(43, 128))) for x in (req.k, req.v))
        q = shift(req.t(np.random.default_rng(4).standard_normal((43, 256)).astype(np.float32)))
        off, lengths, tables = (shift(x) for x in req.batch())
        rope = ov.Rope(shift(req.t((10000.0 ** (-np.arange(32) / 32)).astype(np.float32))), style)
        turned = ov.kv_append(req.cache, k, v, off, lengths, tables, q=q, q_out=shift(torch.zeros_like(q)), rope=rope)
        out = ov.attend(req.cache, turned, off, lengths, tables, out=shift(torch.zeros_like(q)))
        few = ov.attend_selected(req.cache, turned, off, lengths, tables, 2, out=shift(torch.zeros_like(q)))
        made.append([turned, out, few, req.cache.key_view().clone(), req.cache.value_view().clone()])
    for a, b in zip(*made):
        assert torch.equal(a, b)


@pytest.mark.parametrize("requests,most", [(65, 1), (300, 1), (1100, 1), (130, 3), (70, 40)])
def test_many_requests(requests, most):
    """More requests than a wave has lanes, in few and many columns."""
    case("many requests", requests, most)
    rng = np.random.default_rng(requests)
    counts = rng.integers(0 if most > 1 else 1, most + 1, requests)
    contexts = rng.integers(0, 200 if requests < 1000 else 60, requests)
    contexts[rng.integers(requests)] = 2500
    req = Requests(ov, rng, "f16", 1, 64, 32, counts.tolist(), contexts.tolist(), sums=True).fill()
    q = rng.standard_normal((req.rows, 128)).astype(np.float32)
    want, err = attention(req, q, 2)
    check(ov.attend(req.cache, req.t(q), *req.batch(), max_rows=most), want, err)
    check(ov.attend(req.cache, req.t(q), *req.batch()), want, err)
    pages = choose(req, q, 2, 4)
    want, err = attention(req, q, 2, keep=lambda row, a, seen: np.isin(seen // 32, pages[row, a]))
    got = torch.empty(req.rows, 1, 4, dtype=torch.int32, device=DEV)
    check(ov.attend_selected(req.cache, req.t(q), *req.batch(), 4, pages=got), want, err)
    assert np.array_equal(got.cpu().numpy(), pages)


@pytest.mark.parametrize("kv_heads,counts,contexts,window", [
    (64, (1, 200, 64, 90), (100, 0, 300, 17), 0),   # tiles by the place of their last column: as many as the chip holds
    (64, (1, 200, 64, 90), (100, 0, 300, 17), 70),
    (64, (130, 1), (0, 9000), 0),                   # a long one among them, cut
    (128, (1, 1, 1, 1, 1, 1), (9, 80, 200, 1000, 0, 31), 0),
    (1, (700,), (1500,), 0),
    (1, (700,), (1500,), 400),
])
def test_whole_tiles_and_pieces(kv_heads, counts, contexts, window):
    case("tiles", kv_heads, counts, window)
    rng = np.random.default_rng(kv_heads)
    req = Requests(ov, rng, "f16", kv_heads, 64, 32, counts, contexts).fill()
    heads = 2 * kv_heads if kv_heads > 1 else 4
    q = rng.standard_normal((req.rows, heads * 64)).astype(np.float32)
    out = ov.attend(req.cache, req.t(q), *req.batch(), window=window)
    few = [0, kv_heads - 1] if kv_heads > 1 else [0]  # two of the key heads
    group = heads // kv_heads
    part = Requests.__new__(Requests)
    part.__dict__.update(req.__dict__, kv_heads=len(few), k=[k[:, few] for k in req.k], v=[v[:, few] for v in req.v])
    pick = lambda x: x.reshape(req.rows, kv_heads, group * 64)[:, few].reshape(req.rows, -1)  # noqa: E731
    want, err = attention(part, pick(q), group * len(few), window=window)
    check(pick(out.cpu().numpy()), want, err)


@pytest.mark.parametrize("type_", ["f16", "i8"])
def test_a_cache_past_4_gib(type_):
    """Pages at its end: offsets that pass 32 bits in blocks and, with wide heads, in sums."""
    kv_heads, dim, page = 32, 256, 256
    pages = (5 << 30) // (page * kv_heads * dim * (4 if type_ == "f16" else 2))
    case("past 4 GiB", type_, pages)
    cache = ov.KvCache(kv_heads, dim, page, pages, {"f16": ov.TYPE_F16, "i8": ov.TYPE_I8}[type_], sums=True)
    assert cache.byte_count > (5 << 30)
    n = 700
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(n, kv_heads * dim, generator=g, device=DEV) for _ in "kv")
    table = i32([[pages - 1, 0, pages - 2]])
    ov.kv_append(cache, k, v, i32([0, n]), i32([n]), table)
    q = torch.randn(2, kv_heads * dim, generator=g, device=DEV)
    out = ov.attend(cache, q, i32([0, 2]), i32([n]), table)
    few = ov.attend_selected(cache, q, i32([0, 2]), i32([n]), table, 3)
    heads = [0, 31]
    req = Requests.__new__(Requests)
    pick = lambda x, rows: x.reshape(rows, kv_heads, dim)[:, heads].cpu().numpy()  # noqa: E731
    req.__dict__.update(dim=dim, kv_heads=2, rows=2, counts=[2], contexts=[n - 2], off=np.array([0, 2]), type_=type_, k=[pick(k, n)], v=[pick(v, n)])
    want, err = attention(req, pick(q, 2).reshape(2, -1), 2)
    check(pick(out, 2), want.reshape(2, 2, dim), err.reshape(2, 2, dim))
    check(pick(few, 2), want.reshape(2, 2, dim), err.reshape(2, 2, dim))
    sums = cache.sum_view()[pages - 1, heads].cpu().numpy()
    assert np.allclose(sums, as_stored(pick(k, n), type_)[:page].sum(0), rtol=1e-6, atol=1e-5)


def test_most_rows():
    """The most rows that a call takes."""
    rows = 65536
    cache = ov.KvCache(1, 8, 256, rows // 256)
    x = torch.randn(rows, 8, device=DEV)
    table = torch.arange(rows // 256, dtype=torch.int32, device=DEV)[None]
    ov.kv_append(cache, x, x, i32([0, rows]), i32([rows]), table)
    assert torch.equal(cache.value_view().reshape(rows, -1)[:, :8].float(), x.half().float())
    off, lengths = torch.arange(rows + 1, dtype=torch.int32, device=DEV), torch.ones(rows, dtype=torch.int32, device=DEV)
    tables = (torch.arange(rows, dtype=torch.int32, device=DEV) % (rows // 256))[:, None].contiguous()
    got = ov.attend(cache, x, off, lengths, tables, max_rows=1)  # each sees the first token of its page alone
    assert torch.allclose(got, x.half().float()[(torch.arange(rows, device=DEV) % (rows // 256)) * 256], rtol=1e-6, atol=1e-7)


def test_threads_and_contexts():
    """Several threads call into one context, and another context works on its own stream meanwhile."""
    rng = np.random.default_rng(5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctxs = [ov.Context(0), ov.Context(0)]
    jobs, failures = [], []
    for ctx, s in zip(ctxs, streams):
        ctx.set_stream(s.cuda_stream)
    for n in range(6):
        ctx = ctxs[n % 2]
        req = Requests(ov, rng, ["f16", "i8", "bf16"][n % 3], 2, 64, 32, [1, 3 + 9 * (n % 2)], [900, 40], sums=True).fill()
        torch.cuda.synchronize()
        # the same cache's contents in this context's own
        cache = ov.KvCache(2, 64, 32, req.pages, req.cache.type_id, sums=True, ctx=ctx)
        for view in ("key_view", "value_view", "sum_view") + (("scale_view",) if req.type_ == "i8" else ()):
            getattr(cache, view)().copy_(getattr(req.cache, view)())
        q = rng.standard_normal((req.rows, 256)).astype(np.float32)
        out = torch.empty(req.rows, 256, device=DEV)
        few = torch.empty(req.rows, 256, device=DEV)
        calls = [ctx.bind_attend_dev(cache, req.t(q), *req.batch(), out), ctx.bind_attend_selected_dev(cache, req.t(q), *req.batch(), 5, few)]
        jobs.append((req, q, out, few, calls))
    torch.cuda.synchronize()

    def work(calls):
        try:
            for _ in range(50):
                for c in calls:
                    c()
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(j[4],)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures
    for req, q, out, few, calls in jobs:
        check(out, *attention(req, q, 4))
        pages = choose(req, q, 4, 5)
        check(few, *attention(req, q, 4, keep=lambda row, a, seen: np.isin(seen // 32, pages[row, a])))
    jobs.clear()
    threads.clear()
    del req, cache, calls, t
    gc.collect()
    for ctx in ctxs:
        ctx.close()
