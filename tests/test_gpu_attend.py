"""Attention over a paged cache (ovfq_attend[_dev]) against the same in 64 bits; tolerances: kvdata.py."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, Requests, attention, case, check  # noqa: E402


def run(type_, heads, kv_heads, dim, page, counts, contexts, window=0, seed=1, hint=True, spread=1.0, scale=None, whole=True):
    case("attend", type_, heads, kv_heads, dim, page, counts, contexts, window)
    rng = np.random.default_rng(seed)
    req = Requests(ov, rng, type_, kv_heads, dim, page, counts, contexts, spread=spread).fill()
    q = rng.standard_normal((req.rows, heads * dim)).astype(np.float32) * np.float32(1.5)
    out = torch.full((req.rows, heads * dim), 7.0, device=DEV)
    ov.attend(req.cache, req.t(q), *req.batch(), out=out, window=window, scale=scale, max_rows=max(counts) if hint else 0)
    want, err = attention(req, q, heads, window=window, scale=scale)
    check(out, want, err, (type_, heads, counts), whole)
    return req, q, out


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("dim", [8, 64, 80, 96, 128, 192, 256])
def test_decode(type_, dim):
    run(type_, 8, 2, dim, 32, [1, 1, 1], [0, 31, 100])


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("dim", [40, 64, 96, 128, 256])
def test_prompts(type_, dim):
    run(type_, 4, 2, dim, 64, [70, 45], [0, 33])


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (16, 1), (17, 1), (32, 1), (33, 1), (71, 1), (40, 8)])
def test_head_groups(heads, kv_heads):
    run("f16", heads, kv_heads, 64, 32, [1, 2], [90, 5])


@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("type_", ["f16", "i8"])
def test_pages(page, type_):
    run(type_, 4, 1, 64, page, [3, 1], [page - 1, 2 * page + 3])


@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 511, 513])
def test_lengths(length):
    run("f16", 4, 1, 128, 64, [1], [length - 1])


@pytest.mark.parametrize("counts,contexts", [
    ((0, 3, 0, 1, 0), (5, 40, 0, 0, 77)),  # requests without new rows, and one of a single token
    ((1,) * 70, tuple(range(70))),          # more requests than lanes
    ((2, 9, 1, 40, 17), (300, 0, 1000, 64, 5)),  # both kernels in one call
    ((5,) * 9, (0, 1, 30, 31, 32, 33, 400, 800, 64)),
    ((1, 1, 8, 1, 1, 40), (500, 0, 700, 3, 90, 200)),  # a request of two 16-column tiles between single rows and many
])
@pytest.mark.parametrize("hint", [True, False])
def test_batches(counts, contexts, hint):
    run("bf16", 8, 2, 64, 32, counts, contexts, hint=hint)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100])
@pytest.mark.parametrize("counts,contexts", [((1, 4), (300, 0)), ((60,), (150,))])
def test_windows(window, counts, contexts):
    run("f16", 4, 2, 64, 32, counts, contexts, window=window)
    run("i8", 4, 2, 64, 32, counts, contexts, window=window)


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("counts,contexts", [((1,), (9000,)), ((4, 4), (5000, 300)), ((50,), (3000,)), ((1, 1, 1), (8191, 16, 2000))])
def test_split_keys(type_, counts, contexts):
    """Long contexts of few rows: the keys are cut over workgroups and joined."""
    run(type_, 4, 2, 64, 64, counts, contexts)
    run(type_, 4, 1, 128, 256, counts, contexts)


@pytest.mark.parametrize("spread", [1e-6, 30.0])
def test_sizes_of_keys(spread):
    """Scores from nothing to several hundred."""
    run("f16", 4, 2, 64, 32, [1, 40], [200, 60], spread=spread, whole=spread < 2)
    run("bf16", 4, 2, 64, 32, [1, 40], [200, 60], spread=spread, whole=spread < 2)
    run("i8", 4, 2, 64, 32, [1, 40], [200, 60], spread=spread, whole=spread < 2)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(scale):
    run("f16", 4, 2, 64, 32, [2, 40], [100, 0], scale=scale)


@pytest.mark.parametrize("factor", [1e-30, 1e30])
def test_sizes_of_queries(factor):
    """A row's queries are scaled by a power of two before they are rounded."""
    rng = np.random.default_rng(5)
    req = Requests(ov, rng, "f16", 2, 64, 32, [2, 40], [70, 3]).fill()
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    scale = np.float32(0.125 / factor)
    got = ov.attend(req.cache, req.t(q * np.float32(factor)), *req.batch(), scale=scale)
    want, err = attention(req, (q * np.float32(factor)).astype(np.float64), 4, scale=scale)
    check(got, want, err)


def test_host_arrays():
    rng = np.random.default_rng(6)
    req = Requests(ov, rng, "f16", 2, 64, 32, [3, 40], [70, 3])
    flat = lambda x: np.concatenate(x).reshape(-1, 128)  # noqa: E731
    off = np.concatenate([[0], np.cumsum(req.lengths)]).astype(np.int32)
    ov.kv_append(req.cache, flat(req.k), flat(req.v), off, np.array(req.lengths, np.int32), req.tables)
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    got = ov.attend(req.cache, q, *req.batch(False))
    want, err = attention(req, q, 4)
    check(got, want, err)


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("counts,contexts", [((6,), (37,)), ((60,), (37,))])
def test_hidden_tokens_that_are_not_finite(type_, bad, counts, contexts):
    """A row that does not see a token is not touched by it, whatever it holds; rows that see it are."""
    case("hidden", type_, bad, counts)
    rng = np.random.default_rng(7)
    req = Requests(ov, rng, type_, 2, 64, 32, counts, contexts)
    clean = [req.k[0].copy(), req.v[0].copy()]
    at = contexts[0] + counts[0] // 2  # seen by the later rows only
    req.v[0][at, 0, 5] = bad
    req.k[0][at, 1, 9] = bad
    req.fill()
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    got = ov.attend(req.cache, req.t(q), *req.batch()).cpu().numpy()
    req.k[0], req.v[0] = clean
    want, err = attention(req, q, 4)
    before = np.arange(req.rows) < counts[0] // 2
    check(got[before], want[before], err[before])
    after = got[~before].reshape(-1, 4, 64)
    assert not np.isfinite(after[:, :2, 5]).any()
    assert not np.isnan(bad) or np.isnan(after[:, 2:]).all()  # (a score of -inf is a weight of 0)
    if type_ != "i8":  # (an 8-bit token's scale takes all of its channels along)
        rest = np.delete(np.arange(64), 5)
        w, e = want[~before].reshape(-1, 4, 64), err[~before].reshape(-1, 4, 64)
        check(after[:, :2][:, :, rest], w[:, :2][:, :, rest], e[:, :2][:, :, rest])


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
def test_a_page_s_former_tokens(type_):
    """What a page held behind a request's last token, and whole pages that are not its own, count for nothing."""
    rng = np.random.default_rng(8)
    req = Requests(ov, rng, type_, 2, 64, 32, [2, 40], [5, 30])
    bad = np.full((req.pages * 32, 128), np.nan, np.float32)
    everywhere = np.arange(req.pages, dtype=np.int32)[None]
    ov.kv_append(req.cache, req.t(bad), req.t(bad), req.t(np.array([0, len(bad)], np.int32)), req.t(np.array([len(bad)], np.int32)),
                 req.t(everywhere))
    req.fill()
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    want, err = attention(req, q, 4)
    check(ov.attend(req.cache, req.t(q), *req.batch()), want, err)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_queries_that_are_not_finite(bad):
    rng = np.random.default_rng(9)
    req = Requests(ov, rng, "f16", 1, 64, 32, [3, 40], [50, 0]).fill()
    q = rng.standard_normal((req.rows, 2, 64)).astype(np.float32)
    want, err = attention(req, q, 2)
    q[1, 0, 3] = q[20, 1, 60] = bad
    got = ov.attend(req.cache, req.t(q.reshape(req.rows, -1)), *req.batch()).cpu().numpy().reshape(req.rows, 2, 64)
    hit = np.zeros((req.rows, 2), bool)
    hit[1, 0] = hit[20, 1] = True
    assert np.isnan(got[hit]).all()
    check(got[~hit], want.reshape(-1, 2, 64)[~hit], err.reshape(-1, 2, 64)[~hit])


def test_pages_outside_the_cache():
    """Tokens in them are hidden; a row that sees none gives 0."""
    rng = np.random.default_rng(10)
    req = Requests(ov, rng, "f16", 2, 64, 32, [2, 40, 1], [100, 60, 40]).fill()
    lost = {0: [1], 1: [0, 2], 2: [0, 1]}
    for r, entries in lost.items():
        req.tables[r, entries] = [-1, req.pages, 1 << 30][:len(entries)]
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    of = np.repeat(np.arange(3), req.counts)
    want, err = attention(req, q, 4, keep=lambda row, a, seen: ~np.isin(seen // 32, lost[int(of[row])]))
    got = ov.attend(req.cache, req.t(q), *req.batch())
    check(got, want, err)
    assert not got[-1].any()


def test_rows_left_alone():
    """Rows of no request, of requests whose offsets fall or leave the rows, and of more rows than max_rows stay as they were."""
    rng = np.random.default_rng(11)
    req = Requests(ov, rng, "f16", 2, 64, 32, [1, 2, 1, 3], [30, 10, 8, 70]).fill()
    q = rng.standard_normal((9, 4 * 64)).astype(np.float32)
    out = torch.full((9, 4 * 64), 7.0, device=DEV)
    off, lengths, tables = req.batch()
    ov.attend(req.cache, req.t(q), off, lengths, tables, out=out, max_rows=2)
    req.rows = 7
    want, err = attention(req, q[:7], 4)
    check(out[:4], want[:4], err[:4])
    assert (out[4:] == 7).all()
    for broken in ([0, 1, 3, 2, 99], [0, 1, 3, -4, 7]):
        out.fill_(7)
        ov.attend(req.cache, req.t(q), req.t(np.array(broken, np.int32)), lengths, tables, out=out)
        check(out[:3], want[:3], err[:3])
        assert (out[3:] == 7).all()


def test_tokens_before_the_first():
    """A length below the request's rows: the first rows have no token, and give 0."""
    rng = np.random.default_rng(12)
    req = Requests(ov, rng, "f16", 2, 64, 32, [5], [0]).fill()
    q = rng.standard_normal((5, 4 * 64)).astype(np.float32)
    off, lengths, tables = req.batch()
    got = ov.attend(req.cache, req.t(q), off, req.t(np.array([3], np.int32)), tables)
    assert not got[:2].any()
    req.rows, req.counts, req.off = 3, [3], np.array([0, 3], np.int32)
    want, err = attention(req, q[2:], 4)
    check(got[2:], want, err)
    assert not ov.attend(req.cache, req.t(q), off, req.t(np.array([-(1 << 31)], np.int32)), tables).any()


@pytest.mark.parametrize("counts,contexts", [((1, 1, 1), (700, 30, 64)), ((3, 50), (900, 10))])
def test_captured(counts, contexts):
    """One graph serves other lengths and pages on its replays; eager work of the same context lies between them."""
    rng = np.random.default_rng(13)
    ctx, stream = ov.default_context(), torch.cuda.Stream()
    reqs = [Requests(ov, rng, "f16", 2, 64, 64, counts, contexts).fill(), Requests(ov, rng, "f16", 2, 64, 64, counts, contexts[::-1]).fill()]
    # both in the first one's cache: its pages, then the other's
    both = ov.KvCache(2, 64, 64, reqs[0].pages + reqs[1].pages)
    both.key_view()[:reqs[0].pages].copy_(reqs[0].cache.key_view())
    both.key_view()[reqs[0].pages:].copy_(reqs[1].cache.key_view())
    both.value_view()[:reqs[0].pages].copy_(reqs[0].cache.value_view())
    both.value_view()[reqs[0].pages:].copy_(reqs[1].cache.value_view())
    reqs[1].tables = np.where(reqs[1].tables >= 0, reqs[1].tables + reqs[0].pages, -1).astype(np.int32)
    width = max(r.width for r in reqs)
    pad = lambda t: np.pad(t, ((0, 0), (0, width - t.shape[1])), constant_values=-1)  # noqa: E731
    q = rng.standard_normal((reqs[0].rows, 4 * 64)).astype(np.float32)
    qd, out = reqs[0].t(q), torch.empty(reqs[0].rows, 256, device=DEV)
    off, lengths, _ = reqs[0].batch()
    tables = reqs[0].t(pad(reqs[0].tables))
    call = ctx.bind_attend_dev(both, qd, off, lengths, tables, out)
    call()
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for turn in range(4):
            r = reqs[turn % 2]
            lengths.copy_(torch.tensor(r.lengths, dtype=torch.int32))
            tables.copy_(torch.from_numpy(pad(r.tables)))
            out.fill_(7)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want, err = attention(r, q, 4)
            check(out, want, err, turn)
            replayed = out.clone()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                call()
            torch.cuda.synchronize()
            assert torch.equal(out, replayed)
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


def test_the_same_bits_again():
    req, q, out = run("f16", 8, 2, 128, 64, [1, 1, 40], [4000, 100, 900])
    for _ in range(3):
        assert torch.equal(out, ov.attend(req.cache, req.t(q), *req.batch(), max_rows=40))
