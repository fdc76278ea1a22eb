"""Adapter sets that are made, loaded and destroyed while a stream is captured: the capture stays whole."""
import gc

import numpy as np
import pytest

from qdata import normal
from test_gpu_adapters import check, make_adapter, make_weight

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")

DEV = "cuda:0"
K, N, ROWS = 512, 72, 6


class Work:
    """A context, usually on a stream of its own, a weight, and a set with one adapter."""

    def __init__(self, own_stream=True):
        rng, self.gen = np.random.default_rng(1), torch.Generator().manual_seed(1)
        self.ctx, self.stream = ov.Context(0), torch.cuda.Stream()
        if own_stream:  # else torch's default one
            self.ctx.set_stream(self.stream.cuda_stream)
        self.w = make_weight(rng, "q4k", K, N, self.ctx)
        self.x = normal(rng, (ROWS, K))
        self.xd = torch.from_numpy(self.x).to(DEV)
        self.slots = np.array([0, 1, -1, 1, 0, 2], np.int32)
        self.sd = torch.from_numpy(self.slots).to(DEV)
        self.out = torch.zeros(ROWS, N, device=DEV)
        torch.cuda.synchronize()
        self.base = self.projected(None)

    def set(self):
        return ov.AdapterSet(K, N, 2, 16, ov.TYPE_F16, self.ctx)

    def projected(self, s):
        out = torch.empty(ROWS, N, device=DEV)
        torch.cuda.synchronize()
        self.ctx.bind_adapters_dev([self.w], [s], self.xd, self.sd, [out], rows=ROWS)()
        self.ctx.synchronize()
        return out.cpu().numpy()

    def close(self):
        torch.cuda.synchronize()
        del self.w
        gc.collect()
        self.ctx.close()


def test_on_the_captured_stream():
    t = Work()
    s, gone = t.set(), t.set()
    held = {0: (*make_adapter(t.gen, K, N, 9, ov.TYPE_F16), 0.5), 1: (*make_adapter(t.gen, K, N, 16, ov.TYPE_F16), 2.0)}
    for slot, a in held.items():
        s.load(slot, *a)
    size = gone.byte_count
    call = t.ctx.bind_adapters_dev([t.w], [s], t.xd, t.sd, [t.out], rows=ROWS)
    call()
    torch.cuda.synchronize()
    retired = t.ctx.scratch_bytes()[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=t.stream):
        with pytest.raises(ov.OverfitInvalidOperationError):
            t.set()
        call()
        del gone
        gc.collect()
        with pytest.raises(ov.OverfitInvalidOperationError):
            s.load(0, *held[0])
    assert t.ctx.scratch_bytes()[1] == retired + size
    for _ in range(3):
        t.out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(t.out.cpu().numpy(), t.base, t.x, held, t.slots, "replay")
        assert np.array_equal(t.projected(s).view(np.uint32), t.out.cpu().numpy().view(np.uint32))
    del graph
    t.ctx.release_retired()
    assert t.ctx.scratch_bytes()[1] == 0
    check(t.projected(s), t.base, t.x, held, t.slots, "afterwards")
    del call, s
    t.close()


@pytest.mark.parametrize("own_stream", [True, False])
def test_while_another_stream_is_captured(own_stream):
    t = Work(own_stream)
    gone, v, other = t.set(), torch.ones(1000, device=DEV), torch.cuda.Stream()
    torch.cuda.synchronize()
    retired = t.ctx.scratch_bytes()[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=other):
        v.mul_(2)
        s = t.set()
        held = {0: (*make_adapter(t.gen, K, N, 3, ov.TYPE_F16), 1.5), 1: (*make_adapter(t.gen, K, N, 12, ov.TYPE_F16), -1.0)}
        for slot, a in held.items():
            s.load(slot, *a)
        del gone
        gc.collect()
        v.add_(1)
    assert t.ctx.scratch_bytes()[1] == retired  # freed at once
    check(t.projected(s), t.base, t.x, held, t.slots, "made meanwhile")
    want = 1.0
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = 2 * want + 1
        assert (v == want).all()
    del s
    t.close()
