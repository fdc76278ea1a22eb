"""The largest numbers of rows that the norm around the residual sum takes and refuses (ovfq_residual_norm_dev)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from overfit_amd import _lib  # noqa: E402

DEV = "cuda:0"


def test_more_rows_than_a_launch_has_threads_for():
    # refused before anything is launched: the planes are never touched
    lib, ctx = _lib.load(), ov.default_context()
    t = torch.zeros(64, device=DEV)
    for rows in ((1 << 28) - 15, 1 << 28, (1 << 31) - 1):
        for call, p in ((lib.ovfq_residual_norm_dev, t.data_ptr()), (lib.ovfq_residual_norm, 4096)):
            assert call(ctx.handle, p, None, rows, 1, None, None, 0, 1.0, None, p + 128, None) == _lib.OVFQ_ERR_RANGE


@pytest.mark.parametrize("rows,k", [((1 << 28) - 16, 1), ((1 << 28) - 19, 4)])
def test_the_most_rows(rows, k):
    y = torch.full((rows * k,), 3.0, device=DEV)
    y[-k:] = -2.0
    h, _ = ov.residual_norm(y, rows, scale=0.5)
    assert (h[:-k] == 1.5).all() and (h[-k:] == -1.0).all()
