"""What selection of pages keeps beside its inputs and outputs, and that rows whose pages are chosen in turns get the same ones; selection
over more pages than a workgroup holds in registers, and over the widest query groups."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, Requests, attention, case, check  # noqa: E402
from test_gpu_attend_selected import choose  # noqa: E402

MB = 1 << 20


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def filled(ctx, kv_heads, dim, page, pages, type_=None):
    cache = ov.KvCache(kv_heads, dim, page, pages, ov.TYPE_F16 if type_ is None else type_, sums=True, ctx=ctx)
    n = pages * page
    g = torch.Generator(device=DEV).manual_seed(7)
    k, v = (torch.randn(n, kv_heads * dim, generator=g, device=DEV) for _ in "kv")
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)[None]
    ov.kv_append(cache, k, v, i32([0, n]), i32([n]), table)
    return cache, table, n, g


@pytest.mark.parametrize("rows,top,wide,most", [
    (500, 3, 65536, 129 * MB),   # 2.1 GB at once
    (500, 1, 65536, 1 * MB),     # no choice to make
    (500, 64, 63, 1 * MB),       # all pages taken
    (40, 3, 64, 1 * MB),
])
def test_scratch_stays_small(rows, top, wide, most):
    case("scratch", rows, top, wide)
    ctx = ov.Context(0)
    cache, table, n, g = filled(ctx, 8, 8, 32, 63)
    tables = torch.full((1, wide), -1, dtype=torch.int32, device=DEV)
    tables[:, :63] = table
    q = torch.randn(rows, 64, generator=g, device=DEV)
    batch = (i32([0, rows]), i32([n]))
    pages = torch.full((rows, 8, top), -9, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    got = ov.attend_selected(cache, q, *batch, tables, top, pages=pages)
    torch.cuda.synchronize()
    live, retired = ctx.scratch_bytes()
    assert live + retired <= most, (live, retired)
    # the same over the pages that there are, in one turn
    want_pages = torch.full_like(pages, -9)
    want = ov.attend_selected(cache, q, *batch, table, top, pages=want_pages)
    assert torch.equal(pages, want_pages) and torch.equal(got, want) and (pages >= -1).all()
    del cache
    ctx.close()


def test_turns_in_a_graph():
    """A captured call of several turns follows lengths and queries."""
    ctx, stream = ov.Context(0), torch.cuda.Stream()
    cache, table, n, g = filled(ctx, 8, 8, 32, 40)
    tables = torch.full((1, 65536), -1, dtype=torch.int32, device=DEV)
    tables[:, :40] = table
    rows, lengths = 100, i32([n])
    q, out, pages = torch.zeros(rows, 128, device=DEV), torch.zeros(rows, 128, device=DEV), torch.zeros(rows, 8, 4, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    call = ctx.bind_attend_selected_dev(cache, q, i32([0, rows]), lengths, tables, 4, out, pages=pages)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for length in (n, 700, n - 33):
        q.normal_(generator=g)
        lengths.fill_(length)
        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        want = out.clone(), pages.clone()
        out.zero_(), pages.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(pages, want[1]) and out.abs().sum(1).min() > 0
    del call, graph, cache
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    ctx.close()


@pytest.mark.parametrize("pages,top", [(2048, 2), (2049, 40), (2300, 2047), (2300, 2300), (4500, 100), (4500, 2500)])
def test_more_pages_than_registers_hold(pages, top):
    """A thread of the choice keeps eight fits, a workgroup 2048; the others are read again in each step. Some fits are equal, some pages
    are not there."""
    case("pages", pages, top)
    rng = np.random.default_rng(pages + top)
    req = Requests(ov, rng, "f16", 1, 8, 32, [2], [32 * pages + 3], sums=True)
    alike = rng.integers(0, pages, pages // 3)
    for e in alike:  # pages of the same keys: the lower ones first
        req.k[0][32 * e:32 * e + 32] = req.k[0][32 * alike[0]:32 * alike[0] + 32]
    n, tables = req.lengths[0], req.t(req.tables)
    for at in range(0, n, 50000):
        upto = min(n, at + 50000)
        ov.kv_append(req.cache, req.t(req.k[0][at:upto].reshape(-1, 8)), req.t(req.v[0][at:upto].reshape(-1, 8)), i32([0, upto - at]), i32([upto]), tables)
    req.tables[0, rng.integers(0, pages, 20)] = -1
    q = rng.standard_normal((2, 16)).astype(np.float32)
    got = torch.full((2, 1, top), -9, dtype=torch.int32, device=DEV)
    out = ov.attend_selected(req.cache, req.t(q), *req.batch(), top, pages=got)
    want = choose(req, q, 2, top)
    assert np.array_equal(got.cpu().numpy(), want)
    o, err = attention(req, q, 2, keep=lambda row, a, seen: np.isin(seen // 32, want[row, a]))
    check(out, o, err)


@pytest.mark.parametrize("heads,dim", [(64, 256), (128, 128), (136, 120), (2048, 8)])
def test_the_widest_groups(heads, dim):
    """heads * dim / kv_heads up to 16384: 64 KiB of queries in a workgroup's LDS."""
    case("group", heads, dim)
    rng = np.random.default_rng(heads)
    req = Requests(ov, rng, "f16", 1, dim, 32, [1, 2], [300, 100], sums=True).fill()
    q = rng.standard_normal((3, heads * dim)).astype(np.float32)
    got = torch.full((3, 1, 4), -9, dtype=torch.int32, device=DEV)
    out = ov.attend_selected(req.cache, req.t(q), *req.batch(), 4, pages=got)
    want = choose(req, q, heads, 4)
    assert np.array_equal(got.cpu().numpy(), want)
    o, err = attention(req, q, heads, keep=lambda row, a, seen: np.isin(seen // 32, want[row, a]))
    check(out, o, err)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 5])
def test_no_number_comes_behind_the_lowest(dim, heads):
    """Of a page that fits by minus infinity and a lower one whose fit is no number, the first is taken."""
    rng = np.random.default_rng(5)
    req = Requests(ov, rng, "f16", 1, dim, 32, [1], [320], sums=True)
    req.k[0][40, 0, 3] = np.nan
    req.k[0][100, 0, 3] = -np.inf
    req.fill()
    q = np.abs(rng.standard_normal((1, heads * dim))).astype(np.float32)
    for top, want in ((9, [0, 2, 4, 5, 6, 7, 8, 9, 10]), (10, [0, 2, 3, 4, 5, 6, 7, 8, 9, 10]), (11, list(range(11)))):
        pages = torch.full((1, 1, top), -9, dtype=torch.int32, device=DEV)
        ov.attend_selected(req.cache, req.t(q), *req.batch(), top, pages=pages)
        assert pages.cpu().numpy()[0, 0].tolist() == want
