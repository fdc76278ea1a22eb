"""Projections with each row's low-rank adapter (ovfq_project_adapters[_dev]) against the projection alone plus the adapters'
products in 64 bits.

The projection itself is pinned bit for bit elsewhere, so the reference here is project_multi's output on the same device plus
scale * B (A x) in fp64. Tolerance of one output, u = 2^-24 (half a step of fp32, relative): A's sums run over the inputs in at
least 32 partial sums that are then joined, so a product passes through at most n = in / 32 + 32 additions; B's through
rank + 8; the scale, the sum with y and y's own bias add a few more:
  u ((n + 4) |scale| sum_j |B_j| sum_k |A_jk x_k| + (rank + 8) |scale| sum_j |B_j s_j| + 4 (|y| + |delta|))
"""
import ctypes
import sys

import numpy as np
import pytest

from qdata import normal, random_q4k_blocks, random_q6k_blocks

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from overfit_amd import _lib  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
ELEMENT = {ov.TYPE_F32: torch.float32, ov.TYPE_F16: torch.float16, ov.TYPE_BF16: torch.bfloat16}


def case(*what):
    print("[case]", *what, flush=True, file=sys.stderr)


def make_weight(rng, kind, k, n, ctx=None):
    if kind == "q8":
        q = rng.integers(-127, 128, size=n * k, dtype=np.int8)
        s = rng.uniform(1e-4, 1e-3, size=n * k // 32).astype(np.float32)
        return ov.Q8Weight(q, s, k, n, ctx)
    make, cls = (random_q4k_blocks, ov.Q4KWeight) if kind == "q4k" else (random_q6k_blocks, ov.Q6KWeight)
    return cls(make(rng, n * k // 256).reshape(-1), k, n, ctx)


def make_adapter(gen, k, n, rank, type_):
    a = (torch.randn(rank, k, generator=gen) / k ** 0.5).to(ELEMENT[type_])
    b = (torch.randn(n, rank, generator=gen) * 0.3).to(ELEMENT[type_])
    return a, b


def expected(base, x, adapters, row_slots):
    """(outputs, tolerances) in 64 bits: base [rows][n], adapters {slot: (a, b, scale)}."""
    y = base.astype(np.float64)
    tol = 4 * U * np.abs(y)
    xd = x.astype(np.float64)
    for slot, (a, b, scale) in adapters.items():
        rows = np.flatnonzero(row_slots == slot)
        if not len(rows):
            continue
        a, b = a.double().numpy(), b.double().numpy()
        rank, k = a.shape
        low = xd[rows] @ a.T
        delta = scale * (low @ b.T)
        y[rows] += delta
        tol[rows] += U * (4 * np.abs(delta) + abs(scale) * (
            (k / 32 + 36) * (np.abs(xd[rows]) @ np.abs(a).T) @ np.abs(b).T + (rank + 8) * np.abs(low) @ np.abs(b).T))
    return y, tol


def check(got, base, x, adapters, row_slots, what):
    y, tol = expected(base, x, adapters, row_slots)
    got = got.reshape(y.shape)
    plain = ~np.isin(row_slots, list(adapters))
    assert np.array_equal(got[plain].view(np.uint32), base[plain].view(np.uint32)), f"{what}: rows without an adapter"
    off = np.abs(got - y) / tol
    assert np.all(off <= 1), f"{what}: {np.max(off):.2f} times the tolerance at {np.unravel_index(np.argmax(off), off.shape)}"


def run_case(kind, k, ns, rows, ranks, type_, bias=False, pattern="mixed", host=False, missing=(), force=None):
    case(kind, k, ns, rows, ranks, type_, bias, pattern, host, missing, force)
    rng = np.random.default_rng(k + rows * 7 + sum(ns) + sum(ranks))
    gen = torch.Generator().manual_seed(rows * 31 + k)
    slots, max_rank = len(ranks) + 1, max(ranks)  # the last slot stays empty
    ws = [make_weight(rng, kind, k, n) for n in ns]
    x = normal(rng, (rows, k))
    biases = [normal(rng, n) for n in ns] if bias else None
    sets, held = [], []
    for i, n in enumerate(ns):
        if i in missing:
            sets.append(None)
            held.append({})
            continue
        s = ov.AdapterSet(k, n, slots, max_rank, type_)
        ads = {}
        for slot, rank in enumerate(ranks):
            a, b = make_adapter(gen, k, n, rank, type_)
            scale = float(np.float32(rng.uniform(-2, 2)))
            if slot % 2:
                s.load(slot, a.to(DEV), b.to(DEV), scale)
            else:
                s.load(slot, a, b, scale)
            ads[slot] = (a, b, scale)
        sets.append(s)
        held.append(ads)
    if pattern == "one":
        row_slots = np.zeros(rows, np.int32)
    elif pattern == "runs":  # requests of several rows each
        row_slots = ((np.arange(rows) * (slots + 1)) // rows - 1).astype(np.int32)
    else:  # every row its own: loaded, empty, negative and past the set
        row_slots = rng.integers(-2, slots + 2, size=rows).astype(np.int32)
    ctx = ov.default_context()
    if force:
        ctx.set_batched_kernel(force)
    try:
        if host:
            base = ov.project_multi(ws, x.reshape(-1), rows, biases)
            got = ov.project_adapters(ws, sets, x.reshape(-1), row_slots, rows, biases)
        else:
            dev = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(DEV)  # noqa: E731
            bd = None if biases is None else [dev(b) for b in biases]
            base = [o.cpu().numpy() for o in ov.project_multi(ws, dev(x), rows, bd)]
            got = [o.cpu().numpy() for o in ov.project_adapters(ws, sets, dev(x), dev(row_slots), rows, bd)]
    finally:
        if force:
            ctx.set_batched_kernel("auto")
    for i, n in enumerate(ns):
        check(got[i], base[i].reshape(rows, n), x, held[i], row_slots, f"weight {i}")


@pytest.mark.parametrize("type_", [ov.TYPE_F32, ov.TYPE_F16, ov.TYPE_BF16])
@pytest.mark.parametrize("kind,k,ns,rows,ranks", [
    ("q4k", 256, (1,), 1, (1,)),            # one output, rank one
    ("q4k", 512, (100, 17), 1, (8, 3)),     # the decode kernel, two jobs
    ("q4k", 2304, (257,), 1, (16,)),
    ("q6k", 768, (130, 33, 65), 2, (4, 16, 7)),
    ("q8", 32, (5,), 1, (2,)),              # one block of inputs
    ("q8", 96, (48, 16), 3, (5, 9)),
    ("q8", 1056, (70,), 7, (17,)),
    ("q4k", 1024, (96, 40), 15, (16, 12, 8)),
    ("q4k", 512, (64, 16, 16), 16, (16,)),
    ("q6k", 256, (300,), 17, (33, 5)),      # past one 16-row tile
    ("q4k", 768, (1030,), 33, (64, 1)),
    ("q4k", 256, (72, 72), 130, (24, 16, 8, 40)),
    ("q8", 160, (90,), 70, (16, 128)),
])
def test_adapters_match_reference(type_, kind, k, ns, rows, ranks):
    run_case(kind, k, ns, rows, ranks, type_)


@pytest.mark.parametrize("pattern", ["one", "runs"])
@pytest.mark.parametrize("kind,k,ns,rows,ranks,type_", [
    ("q4k", 4096, (1024, 256, 256), 5, (16, 8), ov.TYPE_F16),
    ("q4k", 4096, (512, 512), 64, (32, 16), ov.TYPE_BF16),
    ("q6k", 14336, (256,), 7, (64,), ov.TYPE_BF16),
    ("q8", 4096, (640,), 45, (16, 4, 8), ov.TYPE_F32),
    ("q4k", 2048, (2048, 300), 331, (16, 64, 48), ov.TYPE_F16),
    ("q4k", 512, (200,), 600, (256,), ov.TYPE_BF16),
])
def test_adapters_of_requests(pattern, kind, k, ns, rows, ranks, type_):
    run_case(kind, k, ns, rows, ranks, type_, bias=True, pattern=pattern)


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_adapters_host_pointers(rows):
    run_case("q4k", 512, (130, 20), rows, (8, 5), ov.TYPE_F32, bias=True, host=True)


@pytest.mark.parametrize("rows", [1, 4, 50])
def test_adapters_on_some_weights(rows):
    run_case("q6k", 512, (64, 48, 32), rows, (16, 2), ov.TYPE_BF16, missing=(1,))
    run_case("q4k", 512, (64,), rows, (16, 2), ov.TYPE_F16, missing=(0,))


@pytest.mark.parametrize("force", ["small", "tiled", "rows"])
@pytest.mark.parametrize("kind", ["q4k", "q6k", "q8"])
def test_adapters_beside_forced_kernels(kind, force):
    run_case(kind, 1024, (200,), 6, (16, 8), ov.TYPE_F16, bias=True, force=force)


def test_adapters_long_inputs():
    run_case("q4k", 28672, (48,), 3, (16,), ov.TYPE_F16)
    run_case("q4k", 33792, (20,), 1, (8,), ov.TYPE_BF16)


@pytest.mark.parametrize("rows", [1, 6, 40])
def test_a_bad_adapter_stays_with_its_rows(rows):
    # infinities and NaN in one request's adapter reach no other request's outputs
    rng = np.random.default_rng(rows)
    k, n = 512, 96
    w = make_weight(rng, "q4k", k, n)
    s = ov.AdapterSet(k, n, 3, 16, ov.TYPE_F32)
    gen = torch.Generator().manual_seed(3)
    good = make_adapter(gen, k, n, 12, ov.TYPE_F32)
    bad = [t.clone() for t in make_adapter(gen, k, n, 16, ov.TYPE_F32)]
    bad[0][3, 5] = float("nan")
    bad[1][7, 2] = float("inf")
    s.load(0, *bad, 1.0)
    s.load(2, *good, 0.5)
    x = normal(rng, (rows, k))
    slots = np.where(np.arange(rows) % 2, 0, 2).astype(np.int32)
    dev = lambda v: torch.from_numpy(v).to(DEV)  # noqa: E731
    base = ov.project(w, dev(x), rows=rows).cpu().numpy().reshape(rows, n)
    got = ov.project_adapters([w], [s], dev(x), dev(slots), rows)[0].cpu().numpy().reshape(rows, n)
    mine = slots == 2
    check(got[mine], base[mine], x[mine], {2: (*good, 0.5)}, slots[mine], "the good rows")
    assert np.isnan(got[~mine]).all()


def test_slots_are_replaced_and_emptied():
    rng = np.random.default_rng(9)
    gen = torch.Generator().manual_seed(9)
    k, n, rows = 256, 40, 5
    w = make_weight(rng, "q4k", k, n)
    s = ov.AdapterSet(k, n, 4, 16, ov.TYPE_BF16)
    x = normal(rng, (rows, k))
    xd = torch.from_numpy(x).to(DEV)
    slots = np.array([1, 1, 3, 0, 1], np.int32)
    sd = torch.from_numpy(slots).to(DEV)
    base = ov.project(w, xd, rows=rows).cpu().numpy().reshape(rows, n)
    held = {}
    for step, (slot, rank) in enumerate([(1, 16), (3, 2), (1, 3), (1, None), (0, 9), (1, 15)]):
        if rank is None:
            s.unload(slot)
            held.pop(slot)
        else:
            held[slot] = (*make_adapter(gen, k, n, rank, ov.TYPE_BF16), 1.25)
            s.load(slot, *held[slot])
        got = ov.project_adapters([w], [s], xd, sd, rows)[0].cpu().numpy()
        check(got, base, x, held, slots, f"step {step}")


def test_captured_calls_follow_the_slots():
    # one graph serves any assignment and any adapters loaded later; replays between eager calls
    rng = np.random.default_rng(4)
    gen = torch.Generator().manual_seed(4)
    k, n, rows = 512, 120, 20
    w = make_weight(rng, "q4k", k, n)
    s = ov.AdapterSet(k, n, 3, 16, ov.TYPE_F16)
    x = normal(rng, (rows, k))
    xd, out = torch.from_numpy(x).to(DEV), torch.empty(rows * n, device=DEV)
    sd = torch.zeros(rows, dtype=torch.int32, device=DEV)
    base = ov.project(w, xd, rows=rows).cpu().numpy().reshape(rows, n)
    ctx = ov.default_context()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        call = ctx.bind_adapters_dev([w], [s], xd, sd, [out], rows=rows)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
            with pytest.raises(ov.OverfitInvalidOperationError):
                s.unload(0)
        held = {}
        for step in range(4):
            held[step % 3] = (*make_adapter(gen, k, n, 4 * (step + 1), ov.TYPE_F16), 0.75)
            s.load(step % 3, *held[step % 3])
            slots = rng.integers(-1, 3, size=rows).astype(np.int32)
            sd.copy_(torch.from_numpy(slots))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            replayed = out.cpu().numpy()
            check(replayed, base, x, held, slots, f"replay {step}")
            out.zero_()
            torch.cuda.synchronize()
            call()
            torch.cuda.synchronize()
            assert np.array_equal(out.cpu().numpy().view(np.uint32), replayed.view(np.uint32))
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


def test_same_input_gives_the_same_bits():
    rng = np.random.default_rng(12)
    gen = torch.Generator().manual_seed(12)
    k, n, rows = 4096, 512, 24
    w = make_weight(rng, "q4k", k, n)
    s = ov.AdapterSet(k, n, 4, 16, ov.TYPE_F16)
    for slot in range(4):
        s.load(slot, *make_adapter(gen, k, n, 16, ov.TYPE_F16), 1.0)
    x = torch.from_numpy(normal(rng, (rows, k))).to(DEV)
    sd = torch.from_numpy((np.arange(rows) % 5).astype(np.int32)).to(DEV)
    first = ov.project_adapters([w], [s], x, sd, rows)[0]
    for _ in range(3):
        assert torch.equal(ov.project_adapters([w], [s], x, sd, rows)[0], first)


def test_c_entry_refusals():
    lib = _lib.load()
    rng = np.random.default_rng(1)
    ctx, other = ov.Context(0), ov.Context(0)
    w = make_weight(rng, "q4k", 256, 8, ctx)
    sets = [ov.AdapterSet(256, 8, 2, 4, ov.TYPE_F16, ctx), ov.AdapterSet(256, 8, 2, 4, ov.TYPE_BF16, ctx),
            ov.AdapterSet(512, 8, 2, 4, ov.TYPE_F16, ctx), ov.AdapterSet(256, 9, 2, 4, ov.TYPE_F16, ctx),
            ov.AdapterSet(256, 8, 2, 4, ov.TYPE_F16, other)]
    x, y = torch.zeros(512, device=DEV), torch.zeros(64, device=DEV)
    sl = torch.zeros(4, dtype=torch.int32, device=DEV)

    def call(which, rows=2, slots=sl, c=ctx, weights=None):
        n = len(which)
        arr = ctypes.c_void_p * n
        return lib.ovfq_project_adapters_dev(
            c.handle, n, arr(*[w.handle.value] * n), None if which is None else arr(*[s.handle.value if s else None for s in which]),
            x.data_ptr(), rows, slots, None, arr(*[y.data_ptr()] * n))

    at = ctypes.c_void_p(sl.data_ptr())
    assert call([sets[0]], slots=at) == 0
    assert call([sets[0]], slots=None) == _lib.OVFQ_ERR_NULL
    assert call([sets[0]], slots=ctypes.c_void_p(sl.data_ptr() + 2)) == _lib.OVFQ_ERR_SIZE
    assert call([sets[0]], rows=0, slots=at) == _lib.OVFQ_ERR_RANGE
    assert call([sets[0], sets[1]], slots=at) == _lib.OVFQ_ERR_TYPE
    assert call([sets[2]], slots=at) == _lib.OVFQ_ERR_SIZE
    assert call([sets[3]], slots=at) == _lib.OVFQ_ERR_SIZE
    assert call([sets[4]], slots=at) == _lib.OVFQ_ERR_SIZE
    h = ctypes.c_void_p()
    for args, want in [((8, 256, 8, 2, 4), _lib.OVFQ_ERR_TYPE), ((1, 0, 8, 2, 4), _lib.OVFQ_ERR_RANGE),
                       ((1, 250, 8, 2, 4), _lib.OVFQ_ERR_SIZE), ((1, 256, 0, 2, 4), _lib.OVFQ_ERR_RANGE),
                       ((1, 256, 8, 0, 4), _lib.OVFQ_ERR_RANGE), ((1, 256, 8, 2, 257), _lib.OVFQ_ERR_RANGE),
                       ((1, 1 << 22, 8, 2, 256), _lib.OVFQ_ERR_SIZE)]:
        assert lib.ovfq_adapters_create(ctx.handle, *args, ctypes.byref(h)) == want, args
    host = np.zeros(256 * 8, np.float16)
    for slot, rank, want in [(-1, 1, _lib.OVFQ_ERR_RANGE), (2, 1, _lib.OVFQ_ERR_RANGE), (0, 0, _lib.OVFQ_ERR_RANGE),
                             (0, 5, _lib.OVFQ_ERR_RANGE), (0, 4, 0)]:
        assert lib.ovfq_adapters_load(sets[0].handle, slot, host.ctypes.data, host.ctypes.data, rank, 1.0) == want
    # a context outlives its sets
    assert lib.ovfq_ctx_destroy(other.handle) == _lib.OVFQ_ERR_STATE
    del sets, w
    torch.cuda.synchronize()
    other.close()
    ctx.close()
