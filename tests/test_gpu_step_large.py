"""Adapters, norms and verification where offsets pass 32 bits, at the most slots, and called from several threads at once."""
import threading

import numpy as np
import pytest

import test_gpu_adapters as adapters
import test_gpu_norm as norms
import test_gpu_verify as verify
from test_gpu_adapters import DEV, case, make_adapter, make_weight, ov, torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 4, 20, 40])
def test_slots_past_4_gib(rows):
    # 600 slots of A [256][8192] fp32: 5 GB
    case("slots", rows)
    rng, gen = np.random.default_rng(rows), torch.Generator().manual_seed(rows)
    k, n, slots = 8192, 64, 600
    w = make_weight(rng, "q4k", k, n)
    s = ov.AdapterSet(k, n, slots, 256, ov.TYPE_F32)
    held = {i: (*make_adapter(gen, k, n, rank, ov.TYPE_F32), 1.0) for i, rank in ((0, 16), (522, 256), (599, 40))}
    for i, a in held.items():
        s.load(i, *a)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    sl = np.array([(599, 522, 0, 300)[i % 4] for i in range(rows)], np.int32)
    xd, sd = torch.from_numpy(x).to(DEV), torch.from_numpy(sl).to(DEV)
    base = ov.project(w, xd, rows=rows).cpu().numpy().reshape(rows, n)
    got = ov.project_adapters([w], [s], xd, sd, rows)[0].cpu().numpy()
    adapters.check(got, base, x, held, sl, "past 4 GiB")


def test_the_most_slots():
    case("most slots")
    rng, gen = np.random.default_rng(3), torch.Generator().manual_seed(3)
    k, n, rows = 256, 48, 70
    w = make_weight(rng, "q6k", k, n)
    s = ov.AdapterSet(k, n, 4096, 4, ov.TYPE_BF16)
    held = {int(i): (*make_adapter(gen, k, n, 1 + i % 4, ov.TYPE_BF16), 0.5) for i in np.linspace(0, 4095, 50).astype(int)}
    for i, a in held.items():
        s.load(i, *a)
    sl = rng.choice(list(held) + [7, 4096, 65535, 65536, -1], size=rows).astype(np.int32)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    for r in (1, 6, 30, rows):
        xd, sd = torch.from_numpy(x[:r]).to(DEV), torch.from_numpy(sl[:r]).to(DEV)
        base = ov.project(w, xd, rows=r).cpu().numpy().reshape(r, n)
        got = ov.project_adapters([w], [s], xd, sd, r)[0].cpu().numpy()
        adapters.check(got, base, x[:r], held, sl[:r], f"{r} rows")


def test_norm_planes_past_4_gib():
    case("norm planes")
    rows, k = 70000, 16384
    gen = torch.Generator(device=DEV).manual_seed(1)
    y = torch.randn(rows, k, generator=gen, device=DEV)
    h = torch.randn(rows, k, generator=gen, device=DEV)
    rng = np.random.default_rng(1)
    po, pr = (ov.Norm(1 + 0.3 * rng.standard_normal(k).astype(np.float32)) for _ in range(2))
    at = [0, 1, 65535, 65537, rows - 2, rows - 1]
    want = norms.reference(y[at].cpu().numpy(), h[at].cpu().numpy(), po, None, None, 0.5, pr)
    ho, xo = ov.residual_norm(y, rows, h, norms.on_device(po), None, None, 0.5, norms.on_device(pr), h_out=h, x_out=y)
    norms.check(ho.view(rows, k)[at].cpu().numpy(), want[0], want[1], "h")
    norms.check(xo.view(rows, k)[at].cpu().numpy(), want[2], want[3], "x")


def test_logits_past_4_gib():
    # 9000 rows of 128256, the most of them one token each
    case("logits")
    vocab, rows = 128256, 9000
    gen = torch.Generator(device=DEV).manual_seed(2)
    logits = torch.randn(rows, vocab, generator=gen, device=DEV)
    counts = [0] * (rows - 8) + [3, 3]
    off = np.concatenate([[0], np.cumsum(np.array(counts) + 1)]).astype(np.int32)
    requests = len(counts)
    rng = np.random.default_rng(2)
    temperature = np.where(np.arange(requests) < requests - 4, 0.0, 0.7).astype(np.float32)
    last = rng.random(requests).astype(np.float32)
    some = logits[rows - 8:].cpu().numpy()
    tokens = some[[0, 1, 2, 4, 5, 6]].argmax(1).astype(np.int32)
    u = np.array([0, 1e-6, 0.9, 0, 0, 1e-6], np.float32)
    d = lambda v: torch.from_numpy(v).to(DEV)  # noqa: E731
    accepted, got = ov.verify_drafts(logits, vocab, d(off), d(tokens), d(u), d(last), temperature=d(temperature))
    accepted, got = accepted.cpu().numpy(), got.cpu().numpy()
    greedy = requests - 4
    assert np.array_equal(got[:greedy], logits[:greedy].argmax(1).cpu().numpy()) and not accepted[:greedy].any()
    tail = off[greedy:] - off[greedy]
    want = verify.reference(logits[off[greedy]:].cpu().numpy(), tail, tokens, u, last[greedy:], None, temperature[greedy:])
    assert np.array_equal(accepted[greedy:], want[0]) and np.array_equal(got[off[greedy]:], want[1])


def test_threads_on_one_context():
    # host calls of the three kinds from six threads: the scratch is one, the calls take turns
    case("threads")
    rng, gen = np.random.default_rng(5), torch.Generator().manual_seed(5)
    k, n = 512, 96
    w = make_weight(rng, "q4k", k, n)
    s = ov.AdapterSet(k, n, 3, 16, ov.TYPE_F16)
    held = {i: (*make_adapter(gen, k, n, 16 - i, ov.TYPE_F16), 1.0 + i) for i in range(3)}
    for i, a in held.items():
        s.load(i, *a)
    errors = []

    def work(seed):
        try:
            mine = np.random.default_rng(seed)
            for turn in range(8):
                rows = int(mine.integers(1, 40))
                x = mine.standard_normal((rows, k)).astype(np.float32)
                sl = mine.integers(-1, 4, rows).astype(np.int32)
                base = ov.project(w, x.reshape(-1), rows=rows).reshape(rows, n)
                adapters.check(ov.project_adapters([w], [s], x.reshape(-1), sl, rows)[0], base, x, held, sl, f"thread {seed}")
                y, h = mine.standard_normal((2, rows, k)).astype(np.float32)
                po = ov.Norm(mine.standard_normal(k).astype(np.float32))
                want = norms.reference(y, h, po, None, None, 1.0, po)
                ho, xo = ov.residual_norm(y, rows, h, po, pre=po)
                norms.check(ho, want[0], want[1], "h")
                norms.check(xo, want[2], want[3], "x")
                verify.run(*verify.make(mine, (2, 0, 3), 500, bool(turn % 2)), host=True)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
