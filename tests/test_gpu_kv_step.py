"""Steps of a small model over a paged cache put together from the calls they are made of: norms (each head's own among them), q/k/v
projections, the rotation and the new tokens into each layer's cache, attention, the output projection, the LM head and the check of drafted tokens. Every call is held
against its 64-bit form on the inputs it was given; the whole is captured into one graph, and replayed while the requests grow, lose
refused drafts and end, and others take their pages.
"""
from types import SimpleNamespace

import numpy as np
import pytest

import test_gpu_verify as verify
from kvdata import DEV, attention, case, check
from test_gpu_adapters import make_weight, ov, torch
from test_gpu_kv_append import freqs, turned

pytestmark = pytest.mark.gpu

K, HEADS, KV, DIM, VOCAB, PAGE, LAYERS = 512, 8, 2, 64, 1003, 32, 2


class Model:
    """Weights, one cache a layer, buffers of a step of `rows` rows of `requests` requests, and run(): all calls of a step."""

    def __init__(self, ctx, rng, type_, rows, requests, most, pages, width):
        self.ctx, self.rng, self.type_, self.rows, self.requests = ctx, rng, type_, rows, requests
        f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(DEV)  # noqa: E731
        e = lambda *s: torch.empty(s, device=DEV)  # noqa: E731
        i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
        id_ = {"f16": ov.TYPE_F16, "bf16": ov.TYPE_BF16, "i8": ov.TYPE_I8}[type_]
        self.w = [{"q": make_weight(rng, "q4k", K, HEADS * DIM), "k": make_weight(rng, "q4k", K, KV * DIM),
                   "v": make_weight(rng, "q4k", K, KV * DIM), "o": make_weight(rng, "q4k", HEADS * DIM, K)} for _ in range(LAYERS)]
        self.head = make_weight(rng, "q6k", K, VOCAB)
        self.caches = [ov.KvCache(KV, DIM, PAGE, pages, id_, sums=True) for _ in range(LAYERS)]
        self.norm, self.head_norm = ov.Norm(1 + 0.2 * f(K)), ov.Norm(1 + 0.2 * f(DIM))
        self.freq = freqs(DIM // 2, 10000.0)
        self.rope = ov.Rope(torch.from_numpy(self.freq).to(DEV), "halves")
        self.off, self.len, self.tables = i(requests + 1), i(requests), i(requests, width)
        self.h0 = f(rows, K)
        self.b = [{"x": e(rows, K), "h": e(rows, K), "q": e(rows, HEADS * DIM), "k": e(rows, KV * DIM), "v": e(rows, KV * DIM),
                   "turned": e(rows, HEADS * DIM), "att": e(rows, HEADS * DIM), "o": e(rows, K)} for _ in range(LAYERS)]
        self.logits = e(rows, VOCAB)
        self.last = e(rows, K)
        self.tokens, self.u, self.final = i(max(1, rows - requests)), e(max(1, rows - requests)), e(requests)
        self.accepted, self.answer = i(requests), i(rows)
        c, self.calls, h = ctx, [], self.h0
        for n, (w, b, cache) in enumerate(zip(self.w, self.b, self.caches)):
            if n == 0:
                self.calls.append(c.bind_residual_norm_dev(h, rows, pre=self.norm, x_out=b["x"]))
            else:
                self.calls.append(c.bind_residual_norm_dev(self.b[n - 1]["o"], rows, residual=h, pre=self.norm, h_out=b["h"], x_out=b["x"]))
                h = b["h"]
            self.calls += [
                c.bind_multi_dev([w["q"], w["k"], w["v"]], b["x"], [b["q"], b["k"], b["v"]], rows=rows),
                c.bind_residual_norm_dev(b["q"], rows * HEADS, pre=self.head_norm, x_out=b["q"]),  # each head's own norm, in place
                c.bind_residual_norm_dev(b["k"], rows * KV, pre=self.head_norm, x_out=b["k"]),
                c.bind_kv_append_dev(cache, b["k"], b["v"], self.off, self.len, self.tables, q=b["q"], q_out=b["turned"], rope=self.rope),
                c.bind_attend_dev(cache, b["turned"], self.off, self.len, self.tables, b["att"], max_rows=most),
                c.bind_multi_dev([w["o"]], b["att"], [b["o"]], rows=rows)]
        self.calls += [
            c.bind_residual_norm_dev(self.b[-1]["o"], rows, residual=h, pre=self.norm, h_out=torch.empty_like(self.h0), x_out=self.last),
            c.bind_multi_dev([self.head], self.last, [self.logits], rows=rows),
            c.bind_verify_drafts_dev(self.logits, VOCAB, self.off, self.tokens, self.u, self.final, accepted=self.accepted, tokens=self.answer)]
        # what the caches hold, on the host: (layer, request) -> [tokens][kv heads][dim] of keys and values, as rounded
        self.held = {}

    def run(self):
        for call in self.calls:
            call()

    def place(self, counts, contexts, tables):
        """The requests of the next step: `counts` new rows after `contexts` tokens."""
        put = lambda t, v: t.copy_(torch.from_numpy(np.ascontiguousarray(v)).reshape(t.shape))  # noqa: E731
        self.counts, self.contexts = list(counts), list(contexts)
        put(self.off, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        put(self.len, (np.array(counts) + contexts).astype(np.int32))
        put(self.tables, tables)
        self.h0.normal_()
        put(self.u, self.rng.random(len(self.u)).astype(np.float32) * np.float32(0.02))
        put(self.final, self.rng.random(self.requests).astype(np.float32))
        put(self.tokens, self.rng.integers(0, VOCAB, len(self.tokens)).astype(np.int32))

    def stored(self, layer, what, r):
        """Request r's stored tokens of a layer, read from the cache's memory."""
        cache = self.caches[layer]
        view = cache.key_view() if what == "k" else cache.value_view()
        x = view.reshape(cache.pages, PAGE, KV, DIM).float().cpu().numpy()
        if self.type_ == "i8":
            x = (x - 128) * cache.scale_view()[:, :, "kv".index(what)].reshape(cache.pages, PAGE, KV, 1).cpu().numpy()
        t = np.arange(self.counts[r] + self.contexts[r])
        return x[self.tables.cpu().numpy()[r][t // PAGE], t % PAGE].astype(np.float64)

    def check(self):
        n = lambda t: t.cpu().numpy()  # noqa: E731
        place = np.concatenate([np.arange(m, m + c) for m, c in zip(self.contexts, self.counts)])
        pos = np.repeat(place[:, None], DIM // 2, 1)
        off = np.concatenate([[0], np.cumsum(self.counts)])
        shape = SimpleNamespace(kv_heads=KV, dim=DIM, rows=self.rows, off=off, counts=self.counts, contexts=self.contexts)
        half = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "i8": 0.501 / 127}[self.type_]
        for layer, b in enumerate(self.b):
            want, err = turned(n(b["q"]).reshape(self.rows, HEADS, DIM), pos, self.freq, "halves")
            assert (np.abs(n(b["turned"]).reshape(want.shape) - want) <= err).all()
            keys, err = turned(n(b["k"]).reshape(self.rows, KV, DIM), pos, self.freq, "halves")
            stored = [[self.stored(layer, w, r) for w in "kv"] for r in range(self.requests)]
            for r in range(self.requests):
                rows = slice(off[r], off[r + 1])
                for got, x in ((stored[r][0], keys), (stored[r][1], n(b["v"]).reshape(self.rows, KV, DIM).astype(np.float64))):
                    top = np.abs(x[rows]).max(-1, keepdims=True) if self.type_ == "i8" else np.abs(x[rows])
                    assert (np.abs(got[self.contexts[r]:] - x[rows]) <= top * half * 1.001 + err[rows] * 1.01 + 2.0 ** -25).all()
                    # and what was there before stays
                    old = self.held.get((layer, r, got is stored[r][0]))
                    if old is not None:
                        m = min(len(old), self.contexts[r])
                        assert np.array_equal(got[:m], old[:m])
                self.held[layer, r, True], self.held[layer, r, False] = stored[r]
            o, err = attention(shape, n(b["turned"]), HEADS, stored=lambda r: stored[r])
            check(b["att"], o, err, f"layer {layer}")
        drafts = self.rows - self.requests
        accepted, tokens = verify.reference(n(self.logits), n(self.off), n(self.tokens)[:drafts], n(self.u)[:drafts], n(self.final))
        assert np.array_equal(n(self.accepted), accepted) and np.array_equal(n(self.answer), tokens)
        return accepted



@pytest.mark.parametrize("type_", ["f16", "bf16", "i8"])
@pytest.mark.parametrize("counts,contexts", [((1, 1, 1, 1), (0, 31, 100, 500)), ((4, 4, 4), (29, 64, 700)), ((60, 3, 1), (0, 40, 300))])
def test_steps(type_, counts, contexts):
    case("kv steps", type_, counts)
    rng = np.random.default_rng(sum(counts))
    torch.manual_seed(sum(counts))
    ctx, stream = ov.default_context(), torch.cuda.Stream()
    need = [-(-(m + 4 * c + 4) // PAGE) for m, c in zip(contexts, counts)]
    width, pages = max(need) + 2, sum(need) + 3
    model = Model(ctx, rng, type_, sum(counts), len(counts), max(counts), pages, width)
    free = list(rng.permutation(pages))
    tables = np.full((len(counts), width), -1, np.int32)
    for r, k in enumerate(need):
        tables[r, :k] = [free.pop() for _ in range(k)]
    # what the requests have before: straight into every layer's cache
    for cache in model.caches:
        for r, m in enumerate(contexts):
            if m:
                k = torch.randn(m, KV * DIM, device=DEV)
                ov.kv_append(cache, k, k * 0.5, torch.tensor([0, m], dtype=torch.int32, device=DEV),
                             torch.tensor([m], dtype=torch.int32, device=DEV), torch.from_numpy(tables[r:r + 1]).to(DEV))
    now = list(contexts)
    model.place(counts, now, tables)
    model.run()
    torch.cuda.synchronize()
    accepted = model.check()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            model.run()
        for turn in range(4):
            # refused drafts are written over by the next step's tokens
            now = [m + 1 + int(a) for m, a in zip(now, accepted)] if turn < 3 else now
            if turn == 2:  # the first request ends; another one takes its pages
                now[0] = 0
                tables[0, :need[0]] = tables[0, :need[0]][::-1].copy()
                for key in list(model.held):
                    if key[1] == 0:
                        del model.held[key]
            torch.cuda.synchronize()
            model.place(counts, now, tables)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                accepted = model.check()
            replayed = [b["att"].clone() for b in model.b] + [model.logits.clone()]
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                model.run()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip([b["att"] for b in model.b] + [model.logits], replayed))
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
