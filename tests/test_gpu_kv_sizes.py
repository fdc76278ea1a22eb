"""Paged caches at their largest batches and smallest values, and planes that overlap."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from overfit_amd import _lib  # noqa: E402
from kvdata import DEV, Requests, attention, case, check  # noqa: E402
from test_gpu_attend_selected import choose  # noqa: E402


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def test_many_requests_of_many_heads():
    """Tiles by the million: no launch's threads pass 32 bits."""
    requests, kv_heads = 33000, 64
    case("requests", requests, "kv_heads", kv_heads)
    cache = ov.KvCache(kv_heads, 8, 32, 64)
    v = torch.randn(64, kv_heads * 8, device=DEV)
    ov.kv_append(cache, v, v, torch.arange(65, dtype=torch.int32, device=DEV), i32([1] * 64), torch.arange(64, dtype=torch.int32, device=DEV)[:, None].contiguous())
    pages = torch.arange(requests, dtype=torch.int32, device=DEV) % 64
    off, lengths = torch.arange(requests + 1, dtype=torch.int32, device=DEV), torch.ones(requests, dtype=torch.int32, device=DEV)
    q = torch.randn(requests, kv_heads * 8, device=DEV)
    for most in (0, 1):
        got = ov.attend(cache, q, off, lengths, pages[:, None].contiguous(), max_rows=most)  # each sees the first token of its page alone
        assert torch.allclose(got, v.half().float()[pages.long()], rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("counts,contexts", [((1300,), (700,)), ((650, 1, 640), (0, 5000, 900))])
def test_more_tiles_than_joins(counts, contexts):
    """Pieces of more tiles than the workgroups that join them."""
    case("joins", counts)
    rng = np.random.default_rng(8)
    req = Requests(ov, rng, "f16", 8, 64, 64, counts, contexts).fill()
    q = rng.standard_normal((req.rows, 32 * 64)).astype(np.float32)
    out = ov.attend(req.cache, req.t(q), *req.batch()).cpu().numpy()
    heads = [0, 7]
    part = Requests.__new__(Requests)
    part.__dict__.update(req.__dict__, kv_heads=2, k=[k[:, heads] for k in req.k], v=[v[:, heads] for v in req.v])
    pick = lambda x: x.reshape(req.rows, 8, 4 * 64)[:, heads].reshape(req.rows, -1)  # noqa: E731
    check(pick(out), *attention(part, pick(q), 8))


@pytest.mark.parametrize("size", [1e-44, 1e-40, 1e-37, 3e-37, 5e-37, 1e-30])
def test_smallest_values(size):
    """8-bit heads whose scale has no reciprocal are zeros; above, their quants are those of larger ones."""
    rng = np.random.default_rng(9)
    x = (rng.uniform(-1, 1, (40, 64)) * size).astype(np.float32)
    x[:, 3], x[:, 5] = np.float32(size), 0
    cache = ov.KvCache(1, 64, 64, 1, ov.TYPE_I8)
    t = torch.from_numpy(x).to(DEV)
    ov.kv_append(cache, t, t, i32([0, 40]), i32([40]), i32([[0]]))
    keys = cache.key_view().reshape(64, 64)[:40].cpu().numpy().astype(np.float64) - 128
    values = cache.value_view().reshape(64, 64)[:40].cpu().numpy().astype(np.float64) - 128
    scales = cache.scale_view().reshape(2, 2, 32).permute(1, 0, 2).reshape(2, 64, 1)[:, :40].cpu().numpy().astype(np.float64)
    # a quant is off by half a step and the scale's and its reciprocal's roundings over 127 steps; a head of zeros by its values
    bound = np.where(scales > 0, scales * (0.5 + 127 * 3 * 2.0 ** -24), 127 / 2.0 ** 128 * 1.01)
    for got, s, b in ((keys, scales[0], bound[0]), (values, scales[1], bound[1])):
        assert np.all(np.abs(got * s - x) <= b)
        assert np.all(got[:, 5] == 0)
    assert np.all(scales > 0) == (size > 4e-37)


def test_planes_that_overlap():
    cache = ov.KvCache(2, 16, 32, 4, sums=True)
    ctx, lib = cache.context, cache.context.lib
    mem = torch.zeros(1000, device=DEV)
    f = mem.data_ptr()
    off, lengths, table = i32([0, 3]), i32([3]), i32([[0]])
    batch = _lib.KvBatchStruct(1, 1, 0, off.data_ptr(), lengths.data_ptr(), table.data_ptr())
    freq = torch.ones(8, device=DEV)
    rope = _lib.RopeStruct(16, 0, 1, 1.0, freq.data_ptr(), None)
    q_bytes, k_bytes = 3 * 4 * 16 * 4, 3 * 2 * 16 * 4

    def append(k, v, q, out):
        return lib.ovfq_kv_append_dev(ctx.handle, cache.handle, ctypes.byref(batch), k, v, 3, ctypes.byref(rope), None, q, 4, out)

    k, v = f + q_bytes, f + q_bytes + k_bytes
    assert append(k, v, f, f) == _lib.OVFQ_OK
    assert append(k, v, f, f + 4) == _lib.OVFQ_ERR_SIZE
    assert append(k, v, f + 2000, f + 8) == _lib.OVFQ_ERR_SIZE  # into k
    assert append(f + 2000, k, f + 3000, f + 4) == _lib.OVFQ_ERR_SIZE  # into v
    assert append(f + 2000, v, v + k_bytes, f + q_bytes - 4) == _lib.OVFQ_ERR_SIZE
    for out, want in ((f, _lib.OVFQ_ERR_SIZE), (f + q_bytes - 4, _lib.OVFQ_ERR_SIZE), (f + q_bytes, _lib.OVFQ_OK)):
        assert lib.ovfq_attend_dev(ctx.handle, cache.handle, ctypes.byref(batch), f, 3, 4, 1.0, 0, out) == want
        assert lib.ovfq_attend_selected_dev(ctx.handle, cache.handle, ctypes.byref(batch), f, 3, 4, 1.0, 2, out, None) == want
    torch.cuda.synchronize()
    with pytest.raises(ov.OverfitArgumentError):
        ov.attend(cache, mem[:192].view(3, 64), off, lengths, table, out=mem[4:196].view(3, 64))


def test_one_row_without_its_axis():
    """A single row's queries as a vector."""
    cache = ov.KvCache(2, 16, 32, 1)
    rope = ov.Rope(torch.ones(8, device=DEV))
    q = torch.randn(64, device=DEV)
    batch = (i32([0, 1]), i32([5]), i32([[0]]))
    got = ov.kv_append(cache, None, None, *batch, q=q, rope=rope)
    assert got.shape == q.shape and torch.equal(got, ov.kv_append(cache, None, None, *batch, q=q[None], rope=rope)[0])
    assert ov.attend(cache, got, *batch).shape == q.shape


@pytest.mark.parametrize("requests,most", [(129, 2), (1000, 3), (5000, 2)])
def test_requests_past_a_walk(requests, most):
    """So many requests that a row is searched for and items are counted by a launch of its own."""
    case("requests", requests, most)
    rng = np.random.default_rng(requests)
    counts = rng.integers(0, most + 1, requests)
    contexts = rng.integers(0, 40 if requests < 2000 else 20, requests)
    contexts[rng.integers(requests, size=3)] = [1500, 31, 0]
    req = Requests(ov, rng, "f16", 1, 64, 32, counts.tolist(), contexts.tolist(), sums=True)
    # what came before in one call, page by page as it would come, then the new tokens in one
    first = np.concatenate([[0], np.cumsum(contexts)]).astype(np.int32)
    flat = lambda x, new: req.t(np.concatenate([t[c:] if new else t[:c] for t, c in zip(x, contexts)]).reshape(-1, 64))  # noqa: E731
    ov.kv_append(req.cache, flat(req.k, False), flat(req.v, False), req.t(first), req.t(contexts.astype(np.int32)), req.t(req.tables))
    q = rng.standard_normal((req.rows, 128)).astype(np.float32)
    rope = ov.Rope(torch.zeros(32, device=DEV))  # turned by nothing
    same = ov.kv_append(req.cache, flat(req.k, True), flat(req.v, True), *req.batch(), q=req.t(q), rope=rope)
    assert torch.equal(same.cpu(), torch.from_numpy(q))
    want, err = attention(req, q, 2)
    check(ov.attend(req.cache, same, *req.batch(), max_rows=most), want, err)
    check(ov.attend(req.cache, same, *req.batch()), want, err)
    pages = choose(req, q, 2, 2)
    want, err = attention(req, q, 2, keep=lambda row, a, seen: np.isin(seen // 32, pages[row, a]))
    check(ov.attend_selected(req.cache, same, *req.batch(), 2), want, err)


def test_bad_offsets_among_many():
    """An offset past the rows, at a place that the search looks at: its two requests have no rows, the others theirs."""
    requests, rows = 300, 600
    cache = ov.KvCache(1, 8, 32, requests)
    off = torch.arange(0, rows + 1, 2, dtype=torch.int32, device=DEV)
    off[128] = rows + 5
    lengths, tables = torch.full((requests,), 2, dtype=torch.int32, device=DEV), torch.arange(requests, dtype=torch.int32, device=DEV)[:, None].contiguous()
    k, v, q = (torch.randn(rows, 8, device=DEV) for _ in range(3))
    out = torch.full_like(q, 7.0)
    ov.kv_append(cache, k, v, off, lengths, tables, q=q, q_out=out, rope=ov.Rope(torch.zeros(4, device=DEV)))
    gone = slice(254, 258)
    want = q.clone()
    want[gone] = 7.0
    assert torch.equal(out, want)
    stored = cache.value_view().reshape(requests, 32, -1)[:, :2, :8].reshape(rows, 8).float()
    kept = v.half().float()
    kept[gone] = 0
    assert torch.equal(stored, kept)
    out.fill_(7.0)
    ov.attend(cache, q, off, lengths, tables, out=out)
    assert torch.equal(out[gone], torch.full((4, 8), 7.0, device=DEV))
    assert torch.allclose(out[0::2][:127], kept[0::2][:127], rtol=1e-6, atol=1e-7)  # a request's first token sees itself alone
    assert torch.allclose(out[0::2][129:], kept[0::2][129:], rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("kv_heads,counts,contexts,window", [
    (8, (1500,), (0,), 0),               # tiles of one piece, two and three
    (16, (700, 300, 90), (0, 2000, 5), 0),
    (16, (700, 300, 90), (0, 2000, 5), 300),
    (64, (40,) * 20, tuple(range(0, 4000, 200)), 0),
    (2, (33, 70), (9000, 0), 0),         # more pieces than tiles
])
def test_pieces_by_each_tiles_span(kv_heads, counts, contexts, window):
    case("spans", kv_heads, counts, window)
    rng = np.random.default_rng(31)
    req = Requests(ov, rng, "f16", kv_heads, 64, 64, counts, contexts).fill()
    q = rng.standard_normal((req.rows, 2 * kv_heads * 64)).astype(np.float32)
    out = ov.attend(req.cache, req.t(q), *req.batch(), window=window).cpu().numpy()
    heads = [0, kv_heads - 1]
    part = Requests.__new__(Requests)
    part.__dict__.update(req.__dict__, kv_heads=2, k=[k[:, heads] for k in req.k], v=[v[:, heads] for v in req.v])
    pick = lambda x: x.reshape(req.rows, kv_heads, 2 * 64)[:, heads].reshape(req.rows, -1)  # noqa: E731
    check(pick(out), *attention(part, pick(q), 4, window=window))


def test_a_graph_of_many_requests():
    """Both kernels, their items counted on the device: a captured call follows lengths, offsets and tables as they are when it is replayed."""
    rng = np.random.default_rng(41)
    counts = [1] * 199 + [60]
    req = Requests(ov, rng, "bf16", 2, 64, 32, counts, rng.integers(0, 300, 200).tolist(), sums=True).fill()
    off, lengths, tables = req.batch()
    q = req.t(rng.standard_normal((req.rows, 4 * 64)).astype(np.float32))
    out, few = torch.zeros_like(q), torch.zeros_like(q)
    calls = [req.cache.context.bind_attend_dev(req.cache, q, off, lengths, tables, out, max_rows=60),
             req.cache.context.bind_attend_selected_dev(req.cache, q, off, lengths, tables, 3, few, max_rows=60)]

    def run():
        for c in calls:
            c()
    ctx, side = req.cache.context, torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.set_stream(side.cuda_stream)
    try:
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run()
        replays(req, rng, off, lengths, tables, q, out, few, run, graph)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


def replays(req, rng, off, lengths, tables, q, out, few, run, graph):
    order = np.array([60] + [1] * 199)
    batches = [(req.off, req.lengths, req.tables),
               (np.concatenate([[0], np.cumsum(order)]), np.roll(req.lengths, 1), np.roll(req.tables, 1, 0)),
               (req.off, [n - (n > 80) for n in req.lengths], req.tables)]
    for o, n, t in batches * 2:
        for to, x in ((off, o), (lengths, n), (tables, t)):
            to.copy_(torch.from_numpy(np.ascontiguousarray(np.array(x, np.int32))))
        q.normal_()
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        want = out.clone(), few.clone()
        out.zero_(), few.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(few, want[1])
        assert out.abs().sum(1).min() > 0
