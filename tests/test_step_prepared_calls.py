"""Prepared calls of the operators around the projections: what a call points into lives as long as the call (no GPU needed; the
library's functions are stand-ins that are never given work)."""
import ctypes
import gc
import weakref

import pytest

torch = pytest.importorskip("torch")
import overfit_amd as ov  # noqa: E402


class OnDevice(torch.Tensor):
    """Host memory that says it lies on a device."""

    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))


def plane(n, dtype=torch.float32):
    return torch.zeros(n, dtype=dtype).as_subclass(OnDevice)


class Library:
    def __getattr__(self, name):
        def fn(*args):
            raise AssertionError(f"{name} was called")

        fn.__name__ = name
        return fn


class FakeWeight:
    InputSize, OutputSize = 32, 8
    handle = ctypes.c_void_p(16)

    def __init__(self, context):
        self.context = context


def context(device=0):
    ctx = ov.Context.__new__(ov.Context)
    ctx.lib, ctx.handle, ctx.device = Library(), ctypes.c_void_p(16), device
    return ctx


def held(take_away, refs):
    """`refs` alive with their call after its caller has let go of them."""
    take_away()
    gc.collect()
    assert all(r() is not None for r in refs)


def test_a_norm_that_gets_other_weights():
    ctx = context()
    y, out = plane(64), plane(64)
    post, pre = ov.Norm(plane(16), plane(16)), ov.Norm(plane(16))
    refs = [weakref.ref(t) for t in (post.weight, post.bias, pre.weight)]
    call = ctx.bind_residual_norm_dev(y, 4, post=post, pre=pre, x_out=out)

    def other_weights():
        post.weight, post.bias, pre.weight = plane(16), None, None

    held(other_weights, refs)
    del call
    gc.collect()
    assert all(r() is None for r in refs)


def test_lists_that_are_filled_anew():
    ctx = context()
    weights, sets = [FakeWeight(ctx), FakeWeight(ctx)], [None, None]
    biases, outs = [plane(8), plane(8)], [plane(16), plane(16)]
    refs = [weakref.ref(t) for t in biases + outs + weights]
    call = ctx.bind_adapters_dev(weights, sets, plane(64), plane(2, torch.int32), outs, biases, 2)

    def other_buffers():
        biases[:], outs[:], weights[:] = [None, None], [plane(16), plane(16)], []

    held(other_buffers, refs)
    del call


def test_views_of_tensors_that_are_let_go():
    ctx = context()
    logits, off, final = plane(40), plane(2, torch.int32), plane(1)
    tokens, uniforms, accepted, out = plane(3, torch.int32), plane(3), plane(1, torch.int32), plane(4, torch.int32)
    named = {"logits": logits, "off": off, "final": final, "tokens": tokens, "uniforms": uniforms, "accepted": accepted, "out": out}
    refs = [weakref.ref(t) for t in named.values()]
    call = ctx.bind_verify_drafts_dev(logits, 10, off, tokens, uniforms, final, accepted=accepted, tokens=out)
    del logits, off, final, tokens, uniforms, accepted, out
    held(named.clear, refs)
    del call


def test_a_prepared_call_needs_every_output():
    # an output that the call would make for itself reaches nobody
    ctx = context()
    y = plane(64)
    with pytest.raises(ValueError):
        ctx.bind_residual_norm_dev(y, 4, residual=plane(64), pre=ov.Norm(), h_out=plane(64))
    with pytest.raises(ValueError):
        ctx.bind_adapters_dev([FakeWeight(ctx)], [None], plane(64), plane(2, torch.int32), None, rows=2)
    ctx.bind_residual_norm_dev(y, 4, residual=plane(64), h_out=plane(64))
    ctx.bind_residual_norm_dev(y, 4, residual=plane(64), pre=ov.Norm(), x_out=plane(64))


def test_adapters_on_another_context_than_their_weights():
    # not silently on the weights' context and its stream
    ctx, other = context(), context()
    args = ([FakeWeight(ctx)], [None], plane(64), plane(2, torch.int32), [plane(16)])
    with pytest.raises(ov.OverfitArgumentError):
        other.bind_adapters_dev(*args, rows=2)
    ctx.bind_adapters_dev(*args, rows=2)
