"""New tokens into a paged cache (ovfq_kv_append[_dev]) against the rotation in 64 bits.

Tolerances, u = 2^-24: cosine and sine are off by u (and 2^-40), each product and the sum by u: 3 u scale (|a| + |b|) for a turned channel,
then half a step of the cache's type (2^-25 where fp16 is subnormal). 8-bit keys: half of the scale, and 1.5 * 2^-16 of it for the product with
its reciprocal (127 * 3 u). Values are rounded only: equal to the bit.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, DTYPE, U, Requests, case, quantised  # noqa: E402


def freqs(n, base=500000.0):
    return (base ** (-np.arange(n) / max(n, 1))).astype(np.float32)


def turned(x, pos, freq, style, scale=1.0):
    """(turned, tolerance) in 64 bits; x [rows][heads][dim], pos [rows][pairs]."""
    x = x.astype(np.float64)
    half = len(freq)
    # pos * freq in long double, then less its whole turns: exact to 2^-50 for every position
    turns = pos.astype(np.longdouble) * freq.astype(np.longdouble) / (8 * np.arctan(np.longdouble(1)))
    angle = ((turns - np.rint(turns)) * (8 * np.arctan(np.longdouble(1)))).astype(np.float64)
    c, s = np.cos(angle)[:, None] * scale, np.sin(angle)[:, None] * scale
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if style == "pairs" else (slice(0, half), slice(half, 2 * half))
    out, err = x.copy(), np.zeros_like(x)
    out[..., a], out[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    err[..., a] = err[..., b] = (3 * U + 2.0 ** -40) * abs(scale) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, err


def stored(req, r, what):
    """Request r's stored keys or values [tokens][kv_heads][dim] as fp32, from the cache's memory."""
    view = (req.cache.key_view() if what == "k" else req.cache.value_view())
    flat = view.reshape(req.pages, req.page, req.kv_heads, -1).cpu()
    x = flat.float().numpy() - (128 if req.type_ == "i8" else 0)
    if req.type_ == "i8":
        s = req.cache.scale_view()[:, :, "kv".index(what)].reshape(req.pages, req.page, req.kv_heads, 1).cpu().numpy()
        x = x * s
    t = np.arange(req.lengths[r])
    return x[req.tables[r][t // req.page], t % req.page][..., :req.dim]


def check_keys(req, r, first, want, err, raw):
    got = stored(req, r, "k")[first:]
    if req.type_ == "i8":
        top = np.abs(want).max(-1, keepdims=True) + err.max(-1, keepdims=True)
        tol = err + top / 127 * (0.5 + 1.5 * 2.0 ** -16) + np.abs(want) * 4 * U
    else:
        eps = torch.finfo(DTYPE[req.type_]).eps
        tol = err + (np.abs(want) + err) * eps / 2 + (2.0 ** -25 if req.type_ == "f16" else 0)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)


def check_values(req, r, first):
    got, v = stored(req, r, "v")[first:], req.v[r][first:]
    if req.type_ == "i8":
        q, s = quantised(v)
        assert np.array_equal(got, q * s)
    else:
        assert np.array_equal(got, torch.from_numpy(v).to(DTYPE[req.type_]).float().numpy())


def run(type_, heads, kv_heads, dim, page, counts, contexts, style="pairs", rotary=None, scale=1.0, axes=1, in_place=False, host=False,
        seed=1):
    case("append", type_, heads, kv_heads, dim, page, counts, contexts, style, rotary, axes, in_place, host)
    rng = np.random.default_rng(seed)
    req = Requests(ov, rng, type_, kv_heads, dim, page, counts, contexts)
    half = (dim if rotary is None else rotary) // 2
    freq = freqs(half)
    new = lambda x: np.concatenate([v[m:] for v, m in zip(x, contexts)]).reshape(req.rows, -1)  # noqa: E731
    k, v, q = new(req.k), new(req.v), rng.standard_normal((req.rows, heads * dim)).astype(np.float32)
    place = np.concatenate([np.arange(m, m + n) for m, n in zip(contexts, counts)])
    pos = pair = None
    where = np.repeat(place[:, None], half, 1)
    if axes > 1:
        pos = rng.integers(0, 1 << 20, (axes, req.rows)).astype(np.int32)
        pair = rng.integers(0, axes, half).astype(np.int32)
        where = pos[pair].T
    t = (lambda x: x) if host else req.t
    rope = ov.Rope(t(freq), style, scale, None if pair is None else t(pair))
    qd = t(q.copy())
    got = ov.kv_append(req.cache, t(k), t(v), *req.batch(not host), q=qd, q_out=qd if in_place else None, rope=rope,
                       positions=None if pos is None else t(pos))
    want, err = turned(q.reshape(req.rows, heads, dim), where, freq, style, scale)
    got = (got if host else got.cpu().numpy()).reshape(want.shape)
    assert (np.abs(got - want) <= err).all(), np.max(np.abs(got - want) / (err + 1e-300))
    assert np.array_equal(got[..., 2 * half:], q.reshape(want.shape)[..., 2 * half:])
    want, err = turned(k.reshape(req.rows, kv_heads, dim), where, freq, style, scale)
    for r, m in enumerate(contexts):
        rows = slice(req.off[r], req.off[r + 1])
        if counts[r]:
            check_keys(req, r, m, want[rows], err[rows], k)
            check_values(req, r, m)
    return req


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("style", ["pairs", "halves"])
@pytest.mark.parametrize("dim,rotary", [(8, 8), (40, 24), (64, 64), (80, 32), (96, 96), (128, 128), (128, 64), (136, 102), (256, 256), (256, 2)])
def test_types_and_sizes(type_, style, dim, rotary):
    run(type_, 4, 2, dim, 32, [1, 5], [31, 62], style, rotary)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (7, 1), (40, 8), (71, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_heads(heads, kv_heads, in_place):
    run("f16", heads, kv_heads, 64, 64, [2, 3], [0, 100], "halves", in_place=in_place)
    run("i8", heads, kv_heads, 64, 64, [2, 3], [0, 100], "pairs", 40, in_place=in_place)


@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("rows", [1, 31, 33, 255, 256, 257, 700])
def test_rows(page, rows):
    run("bf16", 2, 1, 64, page, [rows], [17])
    run("i8", 2, 1, 64, page, [rows // 2, 0, rows - rows // 2], [0, 9, 300])


@pytest.mark.parametrize("axes", [2, 3, 4])
@pytest.mark.parametrize("style", ["pairs", "halves"])
def test_axes(axes, style):
    run("f16", 4, 2, 128, 64, [70, 3], [5, 64], style, axes=axes)


@pytest.mark.parametrize("scale", [0.5, 1.2079, -1.0])
def test_scales(scale):
    run("f16", 4, 2, 64, 64, [7], [5], scale=scale)


def test_host_arrays():
    run("f16", 4, 2, 64, 64, [7, 1], [5, 70], host=True)
    run("i8", 4, 2, 80, 64, [7, 1], [5, 70], "halves", 32, axes=3, host=True)


@pytest.mark.parametrize("far", [0, 1, 4095, 131071, (1 << 24) + 1, (1 << 31) - 1, -5, -(1 << 31)])
def test_far_positions(far):
    """Queries alone, turned by given positions."""
    cache = ov.KvCache(1, 64, 32, 1)
    rng = np.random.default_rng(3)
    q = rng.standard_normal((3, 128)).astype(np.float32)
    freq = freqs(32, 10000.0)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    got = ov.kv_append(cache, None, None, i32([0, 3]), i32([3]), i32([[0]]), q=torch.from_numpy(q).to(DEV),
                       rope=ov.Rope(torch.from_numpy(freq).to(DEV)), positions=i32([[far] * 3]))
    want, err = turned(q.reshape(3, 2, 64), np.full((3, 32), far), freq, "pairs")
    off = np.abs(got.cpu().numpy().reshape(want.shape) - want)
    assert (off <= err).all(), np.max(off / err)


def test_axes_without_positions():
    """An axis that there is no position of counts as position 0."""
    cache = ov.KvCache(1, 8, 32, 1)
    q = np.arange(1, 9, dtype=np.float32).reshape(1, 8)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    rope = ov.Rope(torch.ones(4, device=DEV), pair_axes=i32([0, 2, -1, 1]))
    got = ov.kv_append(cache, None, None, i32([0, 1]), i32([1]), i32([[0]]), q=torch.from_numpy(q).to(DEV), rope=rope, positions=i32([[3], [5]]))
    want, err = turned(q.reshape(1, 1, 8), np.array([[3, 0, 0, 5]]), np.ones(4, np.float32), "pairs")
    assert (np.abs(got.cpu().numpy().reshape(1, 1, 8) - want) <= err).all()


@pytest.mark.parametrize("type_", ["f16", "i8"])
def test_nothing_else_is_written(type_):
    """Bad pages, tokens past the table or before the first, rows of no request, requests whose offsets fall: nothing is stored for them,
    and the rest of the cache stays as it was."""
    rng = np.random.default_rng(4)
    req = Requests(ov, rng, type_, 2, 64, 32, [2, 3, 2, 4, 1], [30, 31, 0, 60, 3], extra=4)
    one = torch.ones(req.pages * 32, 128, device=DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    ov.kv_append(req.cache, one, one, i32([0, len(one)]), i32([len(one)]), torch.arange(req.pages, dtype=torch.int32, device=DEV)[None])
    before = [req.cache.key_view().clone(), req.cache.value_view().clone()]
    k = torch.randn(req.rows + 3, 128, device=DEV)
    q, q_out = torch.randn(req.rows + 3, 256, device=DEV), torch.full((req.rows + 3, 256), 7.0, device=DEV)
    rope = ov.Rope(torch.from_numpy(freqs(32)).to(DEV))
    tables = req.tables.copy()
    tables[0, 0], tables[1, :] = -1, req.pages  # both of request 0's tokens; request 1's are in its last entry and past the table
    off = np.array([0, 2, 5, 7, 6, 99], np.int32)  # request 3's offsets fall, the last one's leave the rows
    lengths = np.array([32, req.width * 32 + 2, 1, 64, 4], np.int32)  # request 2: its second row is its first token
    ov.kv_append(req.cache, k, k, req.t(off), req.t(lengths), req.t(tables), q=q, q_out=q_out, rope=rope)
    after = [req.cache.key_view(), req.cache.value_view()]
    changed = {"k": set(), "v": set()}
    for name, a, b in zip("kv", after, before):
        flat = (a != b).reshape(req.pages, 32, 2, -1).any(-1).any(-1)
        changed[name] = {(int(p), int(t)) for p, t in flat.nonzero().tolist()}
    want = {(int(tables[2, 0]), 0)}
    assert changed["k"] == want and changed["v"] == want, (changed, want)
    turned_rows = (q_out != 7).any(1).cpu().numpy()
    assert turned_rows[:7].all() and not turned_rows[7:].any()


def test_the_same_token_again():
    """Appending from an earlier token on (refused drafts) replaces what was there."""
    req = run("f16", 2, 1, 64, 32, [5], [29])
    rng = np.random.default_rng(9)
    req.v[0][30:] = rng.standard_normal((4, 1, 64)).astype(np.float32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    flat = req.t(req.v[0][30:].reshape(4, 64))
    ov.kv_append(req.cache, flat, flat, i32([0, 4]), i32([34]), req.t(req.tables))
    check_values(req, 0, 29)


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("page", [32, 256])
@pytest.mark.parametrize("dim", [40, 96, 128, 256])
def test_sums(type_, page, dim):
    """Each full page's sum of stored keys, in 64 bits rounded once, whether it filled up in one call or over several."""
    case("sums", type_, page, dim)
    rng = np.random.default_rng(5)
    counts, contexts = [1, 2 * page + 3, 7], [page - 1, 5, 2 * page - 3]
    req = Requests(ov, rng, type_, 2, dim, page, counts, contexts, sums=True)
    req.fill()
    got = req.cache.sum_view().cpu().numpy()
    for r, n in enumerate(req.lengths):
        k = stored(req, r, "k").astype(np.float64)
        for e in range(n // page):
            want = k[e * page:(e + 1) * page].sum(0)
            # one rounding to fp32, and 2^-52 of the magnitudes for the order of the additions
            tol = np.abs(want) * U + np.abs(k[e * page:(e + 1) * page]).sum(0) * 2.0 ** -44
            assert (np.abs(got[req.tables[r, e]] - want) <= tol).all()
    untouched = sorted(set(range(req.pages)) - {int(req.tables[r, e]) for r, n in enumerate(req.lengths) for e in range(n // page)})
    assert not got[untouched].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite(bad):
    """It stays with its token and head; 8-bit tokens take all of the head's channels along."""
    rng = np.random.default_rng(6)
    for type_ in ("f16", "bf16", "i8"):
        req = Requests(ov, rng, type_, 2, 64, 32, [3], [0])
        req.v[0][1, 0, 7] = req.k[0][1, 1, 9] = bad
        req.fill()
        for name, raw, head in (("v", req.v[0], 0), ("k", req.k[0], 1)):
            got = stored(req, 0, name)
            hit = np.zeros(got.shape, bool)
            hit[1, head] = type_ == "i8" or np.arange(64) == (7 if name == "v" else 9)
            assert not np.isfinite(got[hit]).any() and np.isfinite(got[~hit]).all(), (type_, name)


def test_large_values():
    """fp16 caches overflow to infinity as the type does; bf16 and 8-bit ones hold what fp32 holds."""
    for type_ in ("f16", "bf16", "i8"):
        req = Requests(ov, np.random.default_rng(7), type_, 1, 64, 32, [2], [0])
        req.v[0][...] = np.float32(7e4)
        req.fill()
        got = stored(req, 0, "v")
        assert np.isinf(got).all() if type_ == "f16" else np.allclose(got, 7e4, rtol=2.0 ** -7)
