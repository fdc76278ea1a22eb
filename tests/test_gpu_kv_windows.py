"""Windows of any length over requests that are shorter than their rows, and offsets of more rows than there are."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from kvdata import DEV, Requests, case  # noqa: E402


@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 40, 1 << 30, 1000])
@pytest.mark.parametrize("rows,length,most", [(60, 45, 0), (60, 20, 60), (9, 5, 0), (9, 5, 9), (400, 300, 0)])
def test_windows_longer_than_what_is_there(window, rows, length, most):
    """A row whose place would be before the first token sees none of them, the others all up to theirs: as without a window."""
    case("window", window, rows, length, most)
    rng = np.random.default_rng(61)
    req = Requests(ov, rng, "f16", 2, 64, 32, [rows], [0]).fill()
    q = req.t(rng.standard_normal((rows, 256)).astype(np.float32))
    off, _, tables = req.batch()
    lengths = req.t(np.array([length], np.int32))
    want = ov.attend(req.cache, q, off, lengths, tables, max_rows=most)
    got = ov.attend(req.cache, q, off, lengths, tables, window=window, max_rows=most)
    assert not want[:rows - length].any() and want[rows - length:].abs().sum(1).min() > 0
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-6)


def test_offsets_that_overlap_without_end():
    """Half of 65536 requests have all of the 65536 rows: tiles past 32 bits. The call leaves its rows as they were."""
    rows, requests, heads = 65536, 65536, 128
    case("overlapping", rows, requests, heads)
    cache = ov.KvCache(1, 8, 32, 1)
    off = torch.zeros(requests + 1, dtype=torch.int32, device=DEV)
    off[1::2] = rows
    lengths = torch.full((requests,), 31, dtype=torch.int32, device=DEV)
    tables = torch.zeros(requests, 1, dtype=torch.int32, device=DEV)
    q = torch.ones(rows, heads * 8, device=DEV)
    out = torch.full_like(q, 7.0)
    ov.attend(cache, q, off, lengths, tables, out=out)
    torch.cuda.synchronize()
    assert (out == 7).all()
