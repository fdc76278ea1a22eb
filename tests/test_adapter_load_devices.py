"""Adapters that are loaded from another device than their set's are refused before the library is called (no GPU needed)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
import overfit_amd as ov  # noqa: E402


class On(torch.Tensor):
    """Host memory that says it lies on cuda:<index>."""

    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))


class On1(On):
    index = 1


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def fn(*args):
            self.calls.append(name)
            return 0

        return fn


def loose_set():
    ctx = ov.Context.__new__(ov.Context)
    ctx.lib, ctx.handle, ctx.device = Library(), ctypes.c_void_p(16), 0
    s = ov.AdapterSet.__new__(ov.AdapterSet)
    s.input_size, s.output_size, s.slots, s.max_rank, s.type_id, s._ctx, s.handle = 64, 8, 2, 4, ov.TYPE_F32, ctx, ctypes.c_void_p(0)
    return s


@pytest.mark.parametrize("where_a,where_b", [(On1, On1), (On, On1), (On1, On)])
def test_another_device(where_a, where_b):
    s = loose_set()
    with pytest.raises(ov.OverfitArgumentError):
        s.load(0, torch.zeros(4, 64).as_subclass(where_a), torch.zeros(8, 4).as_subclass(where_b))
    assert not s._ctx.lib.calls


def test_the_set_s_device_and_the_host():
    s = loose_set()
    s.load(0, torch.zeros(4, 64).as_subclass(On), torch.zeros(8, 4).as_subclass(On))
    s.load(1, torch.zeros(4, 64), torch.zeros(8, 4))
    assert s._ctx.lib.calls == ["ovfq_adapters_load_dev", "ovfq_adapters_load"]
