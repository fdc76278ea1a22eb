"""One verification step of a small model put together from the calls it is made of: the norm in front of a block, projections with
each row's adapter, the norms around the residual sums, the LM head and the drafted tokens' check. Every call is held against its
64-bit form on the inputs it was given, and the whole captured into one graph, replayed with other inputs, requests and adapters.
"""
import numpy as np
import pytest

import test_gpu_adapters as adapters
import test_gpu_norm as norms
import test_gpu_verify as verify
from test_gpu_adapters import DEV, case, make_adapter, make_weight, ov, torch

pytestmark = pytest.mark.gpu

K, KV, FF, VOCAB, SLOTS, RANK = 512, 128, 1024, 3001, 4, 24


class Step:
    """The model's weights, adapters and buffers, and run(): all calls of one step on the current stream."""

    def __init__(self, ctx, rng, gen, rows, requests):
        self.ctx, self.rows, self.gen, self.rng = ctx, rows, gen, rng
        f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(DEV)  # noqa: E731
        shapes = {"q": ("q4k", K, K), "k": ("q4k", K, KV), "v": ("q4k", K, KV), "o": ("q4k", K, K), "gate": ("q4k", K, FF),
                  "up": ("q4k", K, FF), "down": ("q6k", FF, K), "head": ("q6k", K, VOCAB)}
        self.shapes = shapes
        self.w = {n: make_weight(rng, kind, k, out) for n, (kind, k, out) in shapes.items()}
        self.sets = {n: ov.AdapterSet(shapes[n][1], shapes[n][2], SLOTS, RANK, ov.TYPE_BF16) for n in shapes if n != "head"}
        self.held = {n: {} for n in self.sets}
        self.norm = [ov.Norm(1 + 0.2 * f(K)) for _ in range(3)]
        self.channel = f(K)
        e = lambda *s: torch.empty(s, device=DEV)  # noqa: E731
        self.embedded, self.slot = f(rows, K), torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.x0, self.h1, self.x1, self.h2, self.x2, self.act = e(rows, K), e(rows, K), e(rows, K), e(rows, K), e(rows, K), e(rows, FF)
        self.out = {n: e(rows, s[2]) for n, s in shapes.items()}
        self.off = torch.zeros(requests + 1, dtype=torch.int32, device=DEV)
        drafts = rows - requests
        self.tokens = torch.zeros(drafts, dtype=torch.int32, device=DEV)
        self.u, self.last = e(drafts), e(requests)
        self.accepted = torch.zeros(requests, dtype=torch.int32, device=DEV)
        self.answer = torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.calls = self.bind()

    def projected(self, names, x):
        return self.ctx.bind_adapters_dev([self.w[n] for n in names], [self.sets[n] for n in names], x, self.slot,
                                          [self.out[n] for n in names], rows=self.rows)

    def bind(self):
        c, r = self.ctx, self.rows
        return [
            c.bind_residual_norm_dev(self.embedded, r, pre=self.norm[0], x_out=self.x0),
            self.projected("qkv", self.x0),
            self.projected("o", self.out["q"]),  # (the attention between them is not part of this)
            c.bind_residual_norm_dev(self.out["o"], r, residual=self.embedded, gate=self.channel, gate_axis="channel", scale=0.5,
                                     pre=self.norm[1], h_out=self.h1, x_out=self.x1),
            self.projected(["gate", "up"], self.x1),
            lambda: torch.mul(torch.nn.functional.silu(self.out["gate"]), self.out["up"], out=self.act),
            self.projected(["down"], self.act),
            c.bind_residual_norm_dev(self.out["down"], r, residual=self.h1, post=self.norm[2], pre=self.norm[0], h_out=self.h2,
                                     x_out=self.x2),
            c.bind_multi_dev([self.w["head"]], self.x2, [self.out["head"]], rows=r),
            c.bind_verify_drafts_dev(self.out["head"], VOCAB, self.off, self.tokens, self.u, self.last, accepted=self.accepted,
                                     tokens=self.answer),
        ]

    def run(self):
        for call in self.calls:
            call()

    def fill(self, counts):
        """Other inputs, drafts and adapters, in place; `counts`: drafts of each request."""
        rng = self.rng
        put = lambda t, v: t.copy_(torch.from_numpy(np.ascontiguousarray(v)))  # noqa: E731
        off = np.concatenate([[0], np.cumsum(np.array(counts) + 1)]).astype(np.int32)
        put(self.off, off)
        put(self.embedded, rng.standard_normal((self.rows, K)).astype(np.float32))
        put(self.slot, np.repeat(rng.integers(-1, SLOTS, len(counts)), np.array(counts) + 1).astype(np.int32))
        for n, s in self.sets.items():
            slot, rank = int(rng.integers(SLOTS)), int(rng.integers(1, RANK + 1))
            self.held[n][slot] = (*make_adapter(self.gen, *self.shapes[n][1:], rank, ov.TYPE_BF16), 0.75)
            s.load(slot, *self.held[n][slot])
        put(self.tokens, rng.integers(0, VOCAB, sum(counts)).astype(np.int32))
        put(self.u, rng.random(sum(counts)).astype(np.float32) * np.float32(1e-3))
        put(self.last, rng.random(len(counts)).astype(np.float32))

    def likely_drafts(self):
        """Drafts that are mostly the target's likeliest tokens, and chances that accept some of them."""
        first = self.out["head"].argmax(1).cpu().numpy().astype(np.int32)
        off = self.off.cpu().numpy()
        rows = np.concatenate([np.arange(a, b - 1) for a, b in zip(off, off[1:])])
        self.tokens.copy_(torch.from_numpy(first[rows]))

    def check(self):
        n = lambda t: t.cpu().numpy()  # noqa: E731
        slot = n(self.slot)
        norm = lambda v: None if v is None else ov.Norm(n(v.weight))  # noqa: E731

        def around(y, h, post, gate, scale, pre, got_h, got_x, what):
            want = norms.reference(n(y), None if h is None else n(h), norm(post), gate, "channel", scale, norm(pre))
            if got_h is not None:
                norms.check(n(got_h), want[0], want[1], what + " h")
            norms.check(n(got_x), want[2], want[3], what + " x")

        def projections(names, x):
            base = ov.project_multi([self.w[i] for i in names], x, self.rows)
            for i, b in zip(names, base):
                adapters.check(n(self.out[i]), n(b).reshape(self.rows, -1), n(x), self.held[i], slot, i)

        around(self.embedded, None, None, None, 1.0, self.norm[0], None, self.x0, "first")
        projections("qkv", self.x0)
        projections("o", self.out["q"])
        around(self.out["o"], self.embedded, None, n(self.channel), 0.5, self.norm[1], self.h1, self.x1, "second")
        projections(["gate", "up"], self.x1)
        projections(["down"], self.act)
        around(self.out["down"], self.h1, self.norm[2], None, 1.0, self.norm[0], self.h2, self.x2, "third")
        accepted, tokens = verify.reference(n(self.out["head"]), n(self.off), n(self.tokens), n(self.u), n(self.last))
        assert np.array_equal(n(self.accepted), accepted) and np.array_equal(n(self.answer), tokens)
        return accepted


@pytest.mark.parametrize("counts", [(4,), (0,), (3, 0, 5, 4, 4), (7,) * 12])
def test_a_step(counts):
    case("step", counts)
    rng = np.random.default_rng(len(counts))
    gen = torch.Generator().manual_seed(len(counts))
    ctx, stream = ov.default_context(), torch.cuda.Stream()
    rows = sum(counts) + len(counts)
    step = Step(ctx, rng, gen, rows, len(counts))
    step.fill(counts)
    step.run()
    step.likely_drafts()
    step.run()
    accepted = step.check()
    assert accepted.sum() > 0 or not sum(counts)
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step.run()
        for turn in range(3):
            step.fill(counts)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                step.check()
            torch.cuda.synchronize()
            replayed = {i: o.clone() for i, o in step.out.items()}
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                step.run()
            torch.cuda.synchronize()
            assert all(torch.equal(o, replayed[i]) for i, o in step.out.items())
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
