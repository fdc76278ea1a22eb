"""Layer norms (ovfq_residual_norm[_dev]) of rows whose mean is large beside their deviations, against the norm in 64 bits.

A row v of mean M and deviation s, D = mean |v - M|, u = 2^-24 (half a step of fp32, relative), t = max(64, k / 1024) + 16 additions
on the way of any element into a sum over the row. The kernels take the mean m in fp32, E = |m - M| <= t u mean |v|, then the mean
of the differences v - m, which are |v - M| + E at most and u of that off, and take it out of the differences once more:
  the second mean is (t + 1) u (D + E) off, a centred element so e = u (2 |v - M| + E) + (t + 1) u (D + E);
  the variance, mean (v - m)^2 less the second mean's square, (t + 7) u (s^2 + E^2) + 2 E (t + 1) u (D + E);
  the output |w| r e + |x| (half the variance's part of s^2 + eps, and 4 u) + 2 u |x + b|.
No term has the offset itself in first order: u E is its second power in u.
"""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")

DEV = "cuda:0"
U = 2.0 ** -24


def dev(v):
    return None if v is None else torch.from_numpy(np.ascontiguousarray(v)).to(DEV)


def reference(v, weight, bias, eps):
    """(norm, tolerance) in 64 bits."""
    v = v.astype(np.float64)
    t = max(64, v.shape[1] / 1024) + 16
    c = v - v.mean(1, keepdims=True)
    E = t * U * np.abs(v).mean(1, keepdims=True)
    D = np.abs(c).mean(1, keepdims=True)
    var = np.square(c).mean(1, keepdims=True)
    e = U * (2 * np.abs(c) + E) + (t + 1) * U * (D + E)
    var_err = (t + 7) * U * (var + E * E) + 2 * E * (t + 1) * U * (D + E)
    r = 1 / np.sqrt(var + eps)
    x = c * r * weight
    return x + bias, np.abs(weight) * r * e + np.abs(x) * (var_err / (var + eps) / 2 + 4 * U) + 2 * U * np.abs(x + bias)


def check(got, want, tol, what):
    off = np.abs(got.cpu().numpy().reshape(want.shape) - want) / (tol + 1e-300)
    assert np.all(off <= 1), f"{what}: {np.max(off):.2f} times the tolerance at {np.unravel_index(np.argmax(off), off.shape)}"


# a width for each kernel: 16, 32 and 64 lanes a row, two to sixteen waves, rows past 16384; 4096 at few and at many rows
@pytest.mark.parametrize("rows,k", [(5, 50), (4, 64), (9, 127), (5, 256), (3, 500), (4, 1000), (4, 2048), (3, 4096), (1030, 4096),
                                    (3, 8191), (2, 16384), (2, 20001)])
@pytest.mark.parametrize("offset", [0.0, 1e3, 1e4, -3e5])
def test_the_mean_is_taken_out_whole(rows, k, offset):
    print("[case]", rows, k, offset, flush=True, file=sys.stderr)
    rng = np.random.default_rng(k + rows)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    v = (rng.standard_normal((rows, k)) + offset).astype(np.float32)
    weight, bias = 1 + np.float32(0.3) * f(k), np.float32(0.2) * f(k)
    n = ov.Norm(dev(weight), dev(bias), 1e-5, "layer")
    want, tol = reference(v, weight.astype(np.float64), bias.astype(np.float64), np.float32(1e-5))
    _, x = ov.residual_norm(dev(v), rows, pre=n)
    check(x, want, tol, "before a block")
    h, _ = ov.residual_norm(dev(v), rows, post=n)
    check(h, want, tol, "after a block")
    if k <= 16384:
        zero = torch.zeros(rows * k, device=DEV)
        h, x = ov.residual_norm(zero, rows, residual=dev(v), pre=n)
        assert np.array_equal(h.cpu().numpy().reshape(v.shape), v)
        check(x, want, tol, "of the sum")


@pytest.mark.parametrize("k", [64, 1500, 16384, 17001])
def test_rows_of_one_value(k):
    # nothing is left beside the mean: the bias, whatever the value
    values = np.array([0.0, 1.0, 12345.678, -3e5, 1e-3], np.float32)
    v = np.repeat(values[:, None], k, 1)
    bias = np.full(k, 0.5, np.float32)
    want, tol = reference(v, np.ones(k), bias.astype(np.float64), np.float32(1e-5))
    _, x = ov.residual_norm(dev(v), len(values), pre=ov.Norm(None, dev(bias), 1e-5, "layer"))
    check(x, want, tol, "x")
