"""Cosines and sines of far positions against their angles in 60 digits.

An angle's turns are exact but for what doubles lose of numbers below one, 2^-50, the polynomials and the product with 2 pi come to 2^-42,
and a cosine or sine is rounded to fp32 once: half a step of its own.
"""
import decimal
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, case  # noqa: E402

TAU = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def remainder(position, freq):
    """position * freq less whole turns, from the exact product."""
    with decimal.localcontext() as c:
        c.prec = 60
        a = decimal.Decimal(int(position)) * decimal.Decimal(float(freq))
        return float(a - TAU * (a / TAU).to_integral_value())


@pytest.mark.parametrize("base", [10000.0, 500000.0, 0.3])
@pytest.mark.parametrize("far", [1, 4097, 1 << 24, (1 << 29) + 12345, (1 << 30) + 98765431, (1 << 31) - 1, -(1 << 31)])
def test_angles_of_far_positions(far, base):
    case("angles", far, base)
    dim, half = 256, 128
    freq = (base ** (-np.arange(half) / half)).astype(np.float32)
    rows = 5
    places = np.clip(far + np.arange(rows) * (1 if far > 0 else 1 << 20), -(1 << 31), (1 << 31) - 1) if far != (1 << 31) - 1 else far - np.arange(rows)
    q = np.zeros((rows, dim), np.float32)
    q[:, :half] = 1  # a pair (1, 0) turns into its cosine and sine
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    got = ov.kv_append(ov.KvCache(1, dim, 32, 1), None, None, i32([0, rows]), i32([rows]), i32([[0]]), q=torch.from_numpy(q).to(DEV),
                       rope=ov.Rope(torch.from_numpy(freq).to(DEV), "halves"), positions=i32(places.tolist())).cpu().numpy()
    angle = np.array([[remainder(p, f) for f in freq] for p in places])
    for part, fn in ((got[:, :half], np.cos), (got[:, half:], np.sin)):
        want = fn(angle)
        step = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64)
        assert np.all(np.abs(part - want) <= 0.5 * step + 2.0 ** -42), np.max((np.abs(part - want) - 0.5 * step) * 2.0 ** 24)
