"""8-bit caches whose value and key scales are anything where a row does not look, and not finite where one does."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, Requests, attention, check  # noqa: E402


def put(req, r, token, which, value):
    """Keys' (0) or values' (1) scale of a request's token."""
    page, at = int(req.tables[r, token // req.page]), token % req.page
    req.cache.scale_view()[page, at // 32, which, at % 32] = value


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38, 1e30, 1e-45, 0.0])
@pytest.mark.parametrize("counts,window", [((3, 2), 0), ((3, 2), 20), ((60, 45), 0), ((60, 45), 20)])
def test_scales_behind_the_last_token(bad, counts, window):
    rng = np.random.default_rng(21)
    req = Requests(ov, rng, "i8", 2, 64, 64, counts, (70, 5)).fill()
    for r, n in enumerate(req.lengths):
        for token in [t for t in range(n, -(-n // 64) * 64)] + [t for t in range(max(n - counts[r] - window + 1, 0) if window else 0)]:
            for which in (0, 1):
                put(req, r, token, which, float(bad))
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    want, err = attention(req, q, 4, window=window)
    for most in (0, max(counts)):
        check(ov.attend(req.cache, req.t(q), *req.batch(), window=window, max_rows=most), want, err)


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38, 1e30])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("rows,context,token", [(4, 60, 61), (4, 60, 3), (60, 10, 40), (60, 100, 131)])
def test_scales_that_some_rows_see(bad, which, rows, context, token):
    rng = np.random.default_rng(22)
    req = Requests(ov, rng, "i8", 2, 64, 32, [rows], [context]).fill()
    q = rng.standard_normal((req.rows, 4 * 64)).astype(np.float32)
    want, err = attention(req, q, 4)
    put(req, 0, token, which, float(bad))
    got = ov.attend(req.cache, req.t(q), *req.batch()).cpu().numpy()
    first = max(token - context, 0)  # the first row that sees it
    check(got[:first], want[:first], err[:first])
    # (a key's infinite scale may be a weight of 0; finite ones make outputs of any size, up to quants of 127 times 3e38, which is infinite)
    if np.isnan(bad) or (np.isinf(bad) and which == 1):
        assert np.isnan(got[first:]).all()
