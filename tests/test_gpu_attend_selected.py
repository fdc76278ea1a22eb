"""Attention over the pages that fit a row's queries best (ovfq_attend_selected[_dev]) against the same in 64 bits: the pages have to be
equal, the attention over them is held to kvdata.py's tolerances."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, Requests, attention, case, check  # noqa: E402


def choose(req, q, heads, top):
    """[rows][kv_heads][top] pages in rising order, then -1, from the cache's sums."""
    sums = req.cache.sum_view().cpu().numpy().astype(np.float64)
    q = q.reshape(req.rows, req.kv_heads, heads // req.kv_heads, req.dim).astype(np.float64)
    out = np.full((req.rows, req.kv_heads, top), -1, np.int32)
    for r in range(len(req.counts)):
        for i in range(req.counts[r]):
            row, own = req.off[r] + i, (req.contexts[r] + i) // req.page
            for a in range(req.kv_heads):
                ok = [e for e in range(own) if 0 <= req.tables[r, e] < req.pages]
                fit = [(q[row, a] @ sums[req.tables[r, e], a]).max() for e in ok]
                best = sorted(range(len(ok)), key=lambda j: (-fit[j], ok[j]))[:top - 1]
                pages = sorted([ok[j] for j in best] + ([own] if 0 <= req.tables[r, own] < req.pages else []))
                out[row, a, :len(pages)] = pages
    return out


def run(type_, heads, kv_heads, dim, page, counts, contexts, top, seed=1, prepare=None):
    case("selected", type_, heads, kv_heads, dim, page, counts, contexts, top)
    rng = np.random.default_rng(seed)
    req = Requests(ov, rng, type_, kv_heads, dim, page, counts, contexts, sums=True)
    for k in req.k:  # pages differ, so that the choice matters
        k += np.repeat(rng.standard_normal((len(k) // page + 1, kv_heads, dim)), page, 0)[:len(k)].astype(np.float32)
    req.fill()
    q = rng.standard_normal((req.rows, heads * dim)).astype(np.float32)
    if prepare:
        prepare(req, q)
    pages = torch.full((req.rows, kv_heads, top), -9, dtype=torch.int32, device=DEV)
    out = ov.attend_selected(req.cache, req.t(q), *req.batch(), top, pages=pages)
    want = choose(req, q, heads, top)
    assert np.array_equal(pages.cpu().numpy(), want), (np.argwhere(pages.cpu().numpy() != want)[:5], pages.cpu().numpy()[:2], want[:2])
    o, err = attention(req, q, heads, keep=lambda row, a, seen: np.isin(seen // page, want[row, a]))
    check(out, o, err, (type_, counts))
    assert torch.equal(out, ov.attend_selected(req.cache, req.t(q), *req.batch(), top))
    return req, q, out


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("dim", [8, 64, 80, 96, 128, 256])
def test_types_and_sizes(type_, dim):
    run(type_, 4, 2, dim, 32, [1, 3], [400, 900], 4)


@pytest.mark.parametrize("top", [1, 2, 3, 16, 17, 64, 100])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_pages(top, page):
    run("f16", 4, 2, 64, page, [1, 2, 1], [15 * page, 16 * page - 1, 40 * page + 7], top)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (5, 1), (17, 1), (40, 1), (16, 8)])
def test_heads(heads, kv_heads):
    run("f16", heads, kv_heads, 64, 32, [2, 1], [700, 300], 5)


@pytest.mark.parametrize("counts,contexts", [((40,), (500,)), ((1,) * 70, tuple(range(0, 700, 10))), ((0, 2, 0), (9, 300, 9)), ((1,), (0,)), ((3,), (31,))])
def test_batches(counts, contexts):
    run("bf16", 4, 2, 64, 32, counts, contexts, 3)


def test_many_pages():
    """More pages than a workgroup scores, and pieces that are joined."""
    run("f16", 4, 1, 64, 32, [1], [20000], 200)
    run("i8", 4, 1, 64, 32, [2], [20000], 33)


def test_equal_fits():
    """Of equal fits the lower page: all keys alike, then all zero, then zero queries."""
    for seed, fill in ((1, 1.5), (2, 0.0)):
        def alike(req, q):
            for k in req.k:
                k[...] = fill
            req.fill()
            q[...] = abs(q)

        req, _, _ = run("f16", 4, 2, 64, 32, [1, 2], [1000, 333], 5, seed, alike)
    run("f16", 4, 2, 64, 32, [1, 2], [1000, 333], 5, 3, lambda req, q: q.fill(0))


def test_pages_outside_the_cache():
    def lose(req, q):
        req.tables[0, [0, 3, 5]] = [-1, req.pages, 1 << 30]
        req.tables[1, 10] = -1  # its own page

    run("f16", 4, 2, 64, 32, [1, 1], [400, 330], 6, 1, lose)


def test_fits_that_are_no_numbers():
    """They come last."""
    rng = np.random.default_rng(3)
    req = Requests(ov, rng, "f16", 1, 64, 32, [1], [320], sums=True)
    req.k[0][40, 0, 3] = np.nan
    req.k[0][100, 0, 3] = np.inf
    req.fill()
    q = np.abs(rng.standard_normal((1, 64))).astype(np.float32)
    pages = torch.empty(1, 1, 4, dtype=torch.int32, device=DEV)
    ov.attend_selected(req.cache, req.t(q), *req.batch(), 4, pages=pages)
    got = pages.cpu().numpy()[0, 0].tolist()
    assert 3 in got and 1 not in got and got[-1] == 10
    pages = torch.empty(1, 1, 10, dtype=torch.int32, device=DEV)
    ov.attend_selected(req.cache, req.t(q), *req.batch(), 10, pages=pages)
    assert 1 not in pages.cpu().numpy()[0, 0].tolist()


def test_rows_left_alone_and_host_arrays():
    rng = np.random.default_rng(4)
    req = Requests(ov, rng, "f16", 2, 64, 32, [2, 3], [300, 100], sums=True).fill()
    q = rng.standard_normal((7, 256)).astype(np.float32)
    out, pages = torch.full((7, 256), 7.0, device=DEV), torch.full((7, 2, 4), -9, dtype=torch.int32, device=DEV)
    ov.attend_selected(req.cache, req.t(q), *req.batch(), 4, out=out, pages=pages, max_rows=2)
    host_pages = np.zeros((5, 2, 4), np.int32)
    host = ov.attend_selected(req.cache, q[:5], *req.batch(False), 4, pages=host_pages)
    assert np.array_equal(out[:2].cpu().numpy(), host[:2]) and (out[2:] == 7).all() and (pages[2:] == -9).all()
    assert np.array_equal(host_pages, choose(req, q[:5], 4, 4)) and np.array_equal(pages[:2].cpu().numpy(), host_pages[:2])


def test_captured():
    rng = np.random.default_rng(5)
    ctx, stream = ov.default_context(), torch.cuda.Stream()
    req = Requests(ov, rng, "f16", 2, 64, 32, [1, 2], [900, 350], sums=True).fill()
    qd, out = torch.empty(3, 256, device=DEV), torch.empty(3, 256, device=DEV)
    pages = torch.empty(3, 2, 5, dtype=torch.int32, device=DEV)
    batch = req.batch()
    call = ctx.bind_attend_selected_dev(req.cache, qd, *batch, 5, out, pages=pages)
    qd.normal_()
    call()
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for turn in range(4):
            q = rng.standard_normal((3, 256)).astype(np.float32)
            qd.copy_(torch.from_numpy(q))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = choose(req, q, 4, 5)
            assert np.array_equal(pages.cpu().numpy(), want)
            o, err = attention(req, q, 4, keep=lambda row, a, seen: np.isin(seen // 32, want[row, a]))
            check(out, o, err, turn)
            replayed = out.clone()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                call()
            torch.cuda.synchronize()
            assert torch.equal(out, replayed)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
