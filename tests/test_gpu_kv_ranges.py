"""Attention where some of the values are far larger than what a row takes from them, and where all are near fp32's ends.

8-bit values' tolerance is kvdata.py's, but for what fp16 cannot hold of a weight: a weight and its token's scale enter the second product
as one number, in two fp16 parts, against a power of two between 2^-15 and 2^-10 of the largest such number of the row. What the parts
lose is 2^-25 of that power at most, so 2^-35 of the largest, times the quants: 2^-34 max(w scale) sum |quant| holds it twice.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import U, Requests, as_stored, attention, case, check, quantised  # noqa: E402
from test_gpu_kv_scales import put  # noqa: E402


def attention_8bit(req, q, heads, scales, rows=None):
    """(out, tolerance) [rows][heads * dim] in 64 bits; scales[r]: the values' scales of request r, [tokens][kv_heads]."""
    dim, hk = req.dim, req.kv_heads
    group, scale = heads // hk, 1 / math.sqrt(dim)
    q = q.reshape(req.rows, heads, dim).astype(np.float64)
    out, err = np.zeros((req.rows, heads, dim)), np.zeros((req.rows, heads, dim))
    for r in range(len(req.counts)):
        k, quants = as_stored(req.k[r], "i8"), quantised(req.v[r])[0].astype(np.float64)
        for i in range(req.counts[r]):
            row, n = req.off[r] + i, req.contexts[r] + i + 1
            for a in range(hk):
                kk, vs, qq = k[:n, a], scales[r][:n, a].astype(np.float64), q[row, a * group:(a + 1) * group]
                s = qq @ kk.T * scale
                ds = scale * (2 ** -23 * np.abs(qq).max(1)[:, None] * np.abs(kk).sum(1) + (3 * dim + 8) * 2 * U * (np.abs(qq) @ np.abs(kk).T))
                ds = ds + 6 * U * np.abs(s) + 8 * U
                # a token's weight by its own score's error and that of the scores that make up the sum
                e = np.exp(s - s.max(1, keepdims=True))
                w = e / e.sum(1, keepdims=True)
                rel = np.expm1(ds + (w * ds).sum(1, keepdims=True) * 2) + 2 ** -22 + 2 * (3 * n + 64) * 2 * U
                vv = quants[:n, a] * vs[:, None]
                h = slice(a * group, (a + 1) * group)
                out[row, h] = w @ vv
                err[row, h] = (w * rel) @ np.abs(vv) + np.abs(out[row, h]) * 2 ** -22
                err[row, h] += 2 ** -34 * (w * vs).max(1)[:, None] * np.abs(quants[:n, a]).sum(0) + 1e-37
    return out.reshape(req.rows, -1), err.reshape(req.rows, -1)


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 24, 2.0 ** 36, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("drop", [2, 12, 25, 60, 300])
@pytest.mark.parametrize("rows,context,token", [
    (1, 63, 5),      # the first block of several
    (1, 70, 69),     # the last one, masked
    (1, 3000, 1500), # joined from pieces
    (5, 90, 88),
    (40, 70, 75),    # among the new tokens
    (60, 100, 3),
    (60, 2000, 700),
])
def test_a_large_value_of_little_weight(size, drop, rows, context, token):
    case("little weight", size, drop, rows, context, token)
    rng = np.random.default_rng(51)
    req = Requests(ov, rng, "i8", 2, 64, 64, [rows], [context])
    u = rng.standard_normal(64).astype(np.float32)
    u *= np.float32(8 / np.linalg.norm(u))
    q = (rng.standard_normal((rows, 4, 64)) * 0.5 + u).astype(np.float32)
    req.k[0] *= np.float32(0.5)
    req.k[0][token] = -u * np.float32(drop / 8)  # its score is about -drop, the others' of the order of 1
    req.fill()
    q = q.reshape(rows, -1)
    scales = quantised(req.v[0])[1][..., 0].copy()
    scales[token] *= np.float32(size)
    put(req, 0, token, 1, req.t(scales[token]))
    want, err = attention_8bit(req, q, 4, [scales])
    check(ov.attend(req.cache, req.t(q), *req.batch(), max_rows=rows), want, err, whole=False)
    check(ov.attend(req.cache, req.t(q), *req.batch()), want, err, whole=False)


@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1e20, 2.6e36])
@pytest.mark.parametrize("rows,context", [(1, 400), (1, 3000), (40, 300)])
def test_scales_near_the_ends(scale, rows, context):
    """All values' scales as small or large as they can be, but for a share of usual ones."""
    rng = np.random.default_rng(52)
    req = Requests(ov, rng, "i8", 1, 64, 64, [rows], [context]).fill()
    q = rng.standard_normal((rows, 128)).astype(np.float32)
    scales = quantised(req.v[0])[1][..., 0].copy()
    for token in range(0, rows + context, 3):
        scales[token] = np.float32(scale)
        put(req, 0, token, 1, float(scales[token, 0]))
    want, err = attention_8bit(req, q, 2, [scales])
    check(ov.attend(req.cache, req.t(q), *req.batch()), want, err, whole=False)


@pytest.mark.parametrize("type_,size", [("bf16", 2.0 ** 110), ("bf16", 2.0 ** 118), ("bf16", 2.0 ** 124), ("bf16", 2.0 ** -90), ("i8", 2.0 ** 110),
                                        ("i8", 2.0 ** 118), ("i8", 2.0 ** 124), ("i8", 2.0 ** -90), ("f16", 2.0 ** 13), ("f16", 2.0 ** -10)])
@pytest.mark.parametrize("rows,context", [(1, 500), (1, 5000), (3, 40), (60, 300)])
def test_values_near_the_ends(type_, size, rows, context):
    """All of a row's values are that large (fp16: of 65504), that small (fp16: above its denormal ones)."""
    rng = np.random.default_rng(53)
    req = Requests(ov, rng, type_, 2, 64, 64, [rows], [context])
    req.v[0] = np.clip(req.v[0], -4, 4) * np.float32(size)
    req.fill()
    q = rng.standard_normal((rows, 4 * 64)).astype(np.float32)
    unit = lambda r: (as_stored(req.k[r], type_), as_stored(req.v[r], type_) / size)  # noqa: E731
    want, err = attention(req, q, 4, stored=unit)
    got = ov.attend(req.cache, req.t(q), *req.batch()).double().cpu().numpy() / size
    check(got, want, err + (2.0 ** -126 / size if size < 1 else 0))


@pytest.mark.parametrize("which,value", [(0, 1e30), (1, 1e30), (1, 2.6e36)])
@pytest.mark.parametrize("rows,context,token", [(4, 60, 61), (4, 60, 3), (60, 10, 40), (60, 100, 131), (1, 2000, 900)])
def test_finite_scales_that_rows_see(which, value, rows, context, token):
    """The rows that see a token whose key or value scale is far above the others'."""
    rng = np.random.default_rng(22)
    req = Requests(ov, rng, "i8", 2, 64, 32, [rows], [context]).fill()
    q = rng.standard_normal((rows, 4 * 64)).astype(np.float32)
    put(req, 0, token, which, value)
    got = ov.attend(req.cache, req.t(q), *req.batch()).cpu().numpy()
    first = max(token - context, 0)  # the first row that sees it
    assert first < rows
    scales = quantised(req.v[0])[1][..., 0].copy()
    if which == 1:
        scales[token] = np.float32(value)
        want, err = attention_8bit(req, q, 4, [scales])
        check(got, want, err, whole=False)
        return
    # a key's: its score is far above or below all others, so the row is the token's value or what is left without it
    plain, err = attention_8bit(req, q, 4, [scales])
    without, err_without = attention(req, q, 4, keep=lambda row, a, seen: seen != token)
    (quants, _), v = quantised(req.k[0]), as_stored(req.v[0], "i8")
    for row in range(rows):
        for h in range(4):
            at, a = slice(h * 64, (h + 1) * 64), h // 2
            if row < first:
                check(got[row, at], plain[row, at], err[row, at], (row, h), whole=False)
                continue
            score = quants[token, a].astype(np.float64) @ q[row, at]
            assert abs(score) > 1  # times 1e30 / 8
            if score > 0:
                check(got[row, at], v[token, a], np.abs(v[token, a]) * 2.0 ** -20, (row, h), whole=False)
            else:
                check(got[row, at], without[row, at], err_without[row, at], (row, h), whole=False)


@pytest.mark.parametrize("value", [np.inf, 3e38])
@pytest.mark.parametrize("rows,context,token", [(4, 60, 61), (4, 60, 3), (60, 10, 40), (60, 100, 131), (1, 2000, 900)])
def test_scores_past_fp32(value, rows, context, token):
    """A key's scale that makes its scores infinite: above all others the row is no number, below it is what is left without the token.
    A score is one as a power of two: past 2^128 / log2(e)."""
    rng = np.random.default_rng(23)
    req = Requests(ov, rng, "i8", 2, 64, 32, [rows], [context]).fill()
    q = rng.standard_normal((rows, 4 * 64)).astype(np.float32)
    put(req, 0, token, 0, value)
    got = ov.attend(req.cache, req.t(q), *req.batch()).cpu().numpy()
    without, err = attention(req, q, 4, keep=lambda row, a, seen: seen != token)
    plain, err_plain = attention(req, q, 4)
    quants, v = quantised(req.k[0])[0], as_stored(req.v[0], "i8")
    for row in range(rows):
        for h in range(4):
            at = slice(h * 64, (h + 1) * 64)
            if row < max(token - context, 0):
                check(got[row, at], plain[row, at], err_plain[row, at], (row, h), whole=False)
                continue
            score = quants[token, h // 2].astype(np.float64) @ q[row, at]
            size = abs(score) * value / 8 * math.log2(math.e) / 2.0 ** 128
            assert abs(score) > 0.1 and not 0.99 < size < 1.01
            if score > 0 and size < 1:
                check(got[row, at], v[token, h // 2], np.abs(v[token, h // 2]) * 2.0 ** -20, (row, h), whole=False)
            elif score > 0:
                assert np.isnan(got[row, at]).all()
            else:
                check(got[row, at], without[row, at], err[row, at], (row, h), whole=False)


@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("rows", [1, 60])
def test_a_query_with_one_large_channel(type_, rows):
    """A query's parts hold it to 2^-23 of its largest channel, which here no key has much of."""
    rng = np.random.default_rng(54)
    req = Requests(ov, rng, type_, 2, 64, 64, [rows], [500])
    req.k[0][..., 7] *= np.float32(1e-3)
    req.fill()
    q = rng.standard_normal((rows, 4, 64)).astype(np.float32)
    q[..., 7] = 1000
    q = q.reshape(rows, -1)
    want, err = attention(req, q, 4)
    check(ov.attend(req.cache, req.t(q), *req.batch()), want, err, whole=False)
