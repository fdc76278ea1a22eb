"""Weights that are made and destroyed while a stream is captured: the capture stays whole."""
import gc

import numpy as np
import pytest

from qdata import normal, random_q4k_blocks, random_q6k_blocks

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")

DEV = "cuda:0"
K, N, ROWS = 512, 72, 6


class Work:
    """A context, usually on a stream of its own and the ways to a weight on it."""

    def __init__(self, own_stream=True):
        self.rng = np.random.default_rng(2)
        self.ctx, self.stream = ov.Context(0), torch.cuda.Stream()
        if own_stream:  # else torch's default one
            self.ctx.set_stream(self.stream.cuda_stream)
        nb = N * K // 256
        self.q4k, self.q6k = random_q4k_blocks(self.rng, nb).reshape(-1), random_q6k_blocks(self.rng, nb).reshape(-1)
        self.quants = self.rng.integers(-127, 128, size=N * K, dtype=np.int8)
        self.scales = self.rng.uniform(1e-4, 1e-3, size=N * K // 32).astype(np.float32)
        self.gguf = np.zeros((N * K // 32, 34), np.uint8)
        self.q4k_dev = torch.from_numpy(self.q4k.copy()).to(DEV)
        self.x = torch.from_numpy(normal(self.rng, (ROWS, K))).to(DEV)
        torch.cuda.synchronize()

    def ways(self):
        experts = np.concatenate([self.q6k] * 3)
        return [lambda: ov.Q4KWeight(self.q4k, K, N, self.ctx), lambda: ov.Q4KWeight(self.q4k_dev, K, N, self.ctx),
                lambda: ov.Q6KWeight(self.q6k, K, N, self.ctx), lambda: ov.Q8Weight(self.quants, self.scales, K, N, self.ctx),
                lambda: ov.load_gguf_tensor(ov.TYPE_Q8_0, self.gguf.reshape(-1), K, N, self.ctx),
                lambda: ov.load_gguf_experts(ov.TYPE_Q6_K, experts, K, N, 3, self.ctx)]

    def projected(self, w):
        out = torch.empty(ROWS, N, device=DEV)
        torch.cuda.synchronize()
        self.ctx.project_dev(w, self.x, out, rows=ROWS)
        self.ctx.synchronize()
        return out


def test_on_the_captured_stream():
    t = Work()
    w, gone, experts = ov.Q4KWeight(t.q4k, K, N, t.ctx), t.ways()[3](), t.ways()[5]()
    size = gone.ByteCount + sum((e.ByteCount + 255) // 256 * 256 for e in experts)
    want, out = t.projected(w), torch.zeros(ROWS, N, device=DEV)
    torch.cuda.synchronize()
    retired = t.ctx.scratch_bytes()[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=t.stream):
        for way in t.ways():
            with pytest.raises(ov.OverfitInvalidOperationError):
                way()
        t.ctx.project_dev(w, t.x, out, rows=ROWS)
        del gone
        experts.pop()
        gc.collect()
        experts.clear()
        gc.collect()
    assert t.ctx.scratch_bytes()[1] == retired + size
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(t.projected(w), want)
    del graph
    t.ctx.release_retired()
    assert t.ctx.scratch_bytes()[1] == 0 and torch.equal(t.projected(w), want)
    del w
    gc.collect()
    t.ctx.close()


@pytest.mark.parametrize("own_stream", [True, False])
def test_while_another_stream_is_captured(own_stream):
    t = Work(own_stream)
    gone, v, other = [way() for way in t.ways()], torch.ones(1000, device=DEV), torch.cuda.Stream()
    want = t.projected(gone[0])
    retired = t.ctx.scratch_bytes()[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=other):
        v.mul_(2)
        made = [way() for way in t.ways()]
        gone.clear()
        gc.collect()
        v.add_(1)
    assert t.ctx.scratch_bytes()[1] == retired  # freed at once
    assert torch.equal(t.projected(made[0]), want) and torch.equal(t.projected(made[1]), want)
    value = 1.0
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        value = 2 * value + 1
        assert (v == value).all()
    del made
    gc.collect()
    t.ctx.close()
