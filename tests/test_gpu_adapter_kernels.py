"""Adapters beside every projection kernel that adds them to its outputs, and beside those that leave them to a launch of their
own: shapes that reach each (decode rows, split, panel, the tiled kernels, the Q8_0 ones), with ranks on both sides of the 16 and 32
that are staged at a time and with more slots than rows share. Reference and tolerance: test_gpu_adapters.py.
"""
import numpy as np
import pytest

from test_gpu_adapters import DEV, case, check, make_adapter, make_weight, ov, run_case, torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = ov.TYPE_F32, ov.TYPE_F16, ov.TYPE_BF16
MANY = tuple(1 + 5 * i % 37 for i in range(24))  # 24 slots of ranks 1 to 37


@pytest.mark.parametrize("kind,k,ns,ranks", [
    ("q4k", 512, (300, 33, 5, 70), (256, 100)),  # two rows a wave
    ("q4k", 4352, (301,), (64, 130)),            # one, eight waves a workgroup
    ("q6k", 768, (100, 3), (31, 256)),
    ("q6k", 256, (65700,), (12,)),               # eight waves for many rows
    ("q8", 512, (129, 40), (200, 33)),
    ("q8", 9216, (65,), (16,)),                  # quantised by a launch of its own
])
@pytest.mark.parametrize("pattern", ["one", "mixed"])
def test_one_row(kind, k, ns, ranks, pattern):
    run_case(kind, k, ns, 1, ranks, BF16, bias=True, pattern=pattern)


@pytest.mark.parametrize("rows", [2, 3, 5, 8])
@pytest.mark.parametrize("kind,k,ns,ranks", [
    ("q4k", 1024, (200, 33, 65), MANY),
    ("q4k", 3840, (90, 50, 20), (8, 70)),
    ("q6k", 512, (130, 17, 40), (33, 256)),
    ("q6k", 2048, (40, 65, 30, 20), (256, 1)),  # products past the kernel's LDS
    ("q8", 1024, (200, 31), MANY),
    ("q8", 4096, (97,), (256, 17)),
    ("q8", 4096, (40, 50, 60, 70), (256, 17)),  # past it
])
def test_few_rows(kind, k, ns, ranks, rows):
    run_case(kind, k, ns, rows, ranks, F16, bias=rows % 2 == 1)


@pytest.mark.parametrize("kind,k,ns,rows,ranks", [
    ("q4k", 4096, (512,), 16, MANY),          # split: one to four row tiles, four and eight waves
    ("q4k", 1024, (512, 40, 30), 20, MANY),
    ("q4k", 4096, (1000, 300), 35, (64, 33)),
    ("q4k", 4096, (257,), 64, MANY),
    ("q6k", 4096, (512, 100, 65), 9, (128, 5)),
    ("q6k", 1024, (300, 300), 33, MANY),
    ("q6k", 5120, (300,), 50, (16, 40)),
    ("q4k", 256, (12400,), 10, (16, 40)),     # panel: one to five row tiles
    ("q4k", 512, (12400,), 30, MANY),
    ("q4k", 256, (12350,), 45, (33,)),
    ("q4k", 256, (12400,), 60, MANY),
    ("q4k", 512, (12400, 100), 70, (100, 2)),
    ("q6k", 512, (12400,), 12, (16, 40)),
    ("q6k", 256, (12400,), 30, MANY),
    ("q6k", 256, (12350, 70), 60, (65,)),
    ("q8", 512, (400,), 10, MANY),            # Q8_0 split and panel
    ("q8", 4096, (400, 20), 16, (128, 3)),
    ("q8", 544, (400,), 30, MANY),
    ("q8", 4096, (260,), 31, (16, 70)),
    ("q8", 2048, (8200,), 40, MANY),
    ("q8", 1024, (3000,), 300, (64, 16)),
    ("q8", 512, (100,), 530, (16, 4)),        # past the panel kernel's rows
])
@pytest.mark.parametrize("pattern", ["mixed", "runs"])
def test_batches(kind, k, ns, rows, ranks, pattern):
    run_case(kind, k, ns, rows, ranks, F32 if rows % 3 == 0 else BF16, bias=True, pattern=pattern)


@pytest.mark.parametrize("kind,k,ns,rows,ranks", [
    ("q4k", 512, (200, 30), 70, MANY),        # the 64-row kernel
    ("q4k", 256, (130,), 1030, (16, 40, 8)),  # its 128-row form
    ("q4k", 256, (14336,), 130, MANY),        # wide
    ("q4k", 512, (7200, 7200), 140, (48, 16)),
    ("q4k", 768, (6400,), 200, MANY),         # pair
    ("q6k", 768, (1000,), 70, (16, 40, 8)),   # pair
    ("q6k", 768, (6200,), 200, MANY),         # pair-wide
    ("q6k", 512, (6200,), 137, (33, 16)),
    ("q6k", 256, (9000,), 130, (16, 40, 8)),  # the 64-row kernel
    ("q6k", 512, (100,), 1030, MANY),
])
@pytest.mark.parametrize("pattern", ["mixed", "runs", "one"])
def test_tiled(kind, k, ns, rows, ranks, pattern):
    run_case(kind, k, ns, rows, ranks, F16, bias=pattern != "one", pattern=pattern, force="tiled")


@pytest.mark.parametrize("rows", [70, 1030])
def test_prepared_weights(rows):
    rng = np.random.default_rng(rows)
    gen = torch.Generator().manual_seed(rows)
    k, n = 512, 200
    case("prepared", rows)
    w = make_weight(rng, "q6k", k, n)
    w.prepare_mfma()
    s = ov.AdapterSet(k, n, 2, 48, F16)
    held = {i: (*make_adapter(gen, k, n, rank, F16), 0.5 + i) for i, rank in enumerate((48, 7))}
    for i, a in held.items():
        s.load(i, *a)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    slots = rng.integers(-1, 2, size=rows).astype(np.int32)
    xd, sd = torch.from_numpy(x).to(DEV), torch.from_numpy(slots).to(DEV)
    ctx = ov.default_context()
    ctx.set_batched_kernel("tiled")
    try:
        base = ov.project(w, xd, rows=rows).cpu().numpy().reshape(rows, n)
        got = ov.project_adapters([w], [s], xd, sd, rows)[0].cpu().numpy()
    finally:
        ctx.set_batched_kernel("auto")
    check(got, base, x, held, slots, "prepared")


@pytest.mark.parametrize("kind,rows", [("q4k", 1), ("q4k", 3), ("q4k", 24), ("q4k", 70), ("q8", 2), ("q8", 20)])
def test_two_graphs_share_the_scratch(kind, rows):
    # two captured calls of one context and an eager one between: each replay writes what it reads
    rng = np.random.default_rng(rows)
    gen = torch.Generator().manual_seed(rows)
    ctx, stream = ov.default_context(), torch.cuda.Stream()
    calls = []
    for k, ns, rank in ((512, (96, 40), 16), (1024, (200,), 40)):
        case(kind, rows, k)
        ws = [make_weight(rng, kind, k, n) for n in ns]
        sets = [ov.AdapterSet(k, n, 3, rank, BF16) for n in ns]
        held = [{i: (*make_adapter(gen, k, n, rank - i, BF16), 1.5 - i) for i in range(2)} for n in ns]
        for s, h in zip(sets, held):
            for i, a in h.items():
                s.load(i, *a)
        x = rng.standard_normal((rows, k)).astype(np.float32)
        slots = rng.integers(0, 3, size=rows).astype(np.int32)
        xd, sd = torch.from_numpy(x).to(DEV), torch.from_numpy(slots).to(DEV)
        out = [torch.empty(rows * n, device=DEV) for n in ns]
        base = [o.cpu().numpy().reshape(rows, -1) for o in ov.project_multi(ws, xd, rows)]
        calls.append((ws, sets, xd, sd, out, rows, x, slots, held, base))
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graphs = []
        for ws, sets, xd, sd, out, rows, *_ in calls:
            call = ctx.bind_adapters_dev(ws, sets, xd, sd, out, rows=rows)
            call()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                call()
            graphs.append((g, call))
        for turn in range(3):
            for (g, call), (_, _, _, _, out, rows, x, slots, held, base) in zip(graphs, calls):
                for o in out:
                    o.fill_(7.0)
                torch.cuda.synchronize()
                g.replay()
                graphs[turn % 2][1]()
                torch.cuda.synchronize()
                for o, h, b in zip(out, held, base):
                    check(o.cpu().numpy(), b, x, h, slots, f"turn {turn}")
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("slots", [3, 9])
@pytest.mark.parametrize("kind,n,rows,force", [("q4k", 12400, 50, None), ("q4k", 200, 150, "tiled"), ("q4k", 14336, 140, "tiled"),
                                               ("q6k", 6200, 140, "tiled"), ("q8", 3000, 200, None), ("q8", 300, 20, None)])
def test_a_bad_adapter_stays_with_its_rows(kind, n, rows, force, slots):
    # infinities and NaN in one request's adapter reach no other request's outputs, in runs of rows and one beside the other
    case("bad", kind, n, rows, force, slots)
    rng = np.random.default_rng(rows)
    gen = torch.Generator().manual_seed(rows)
    k = 512
    w = make_weight(rng, kind, k, n)
    s = ov.AdapterSet(k, n, slots, 40, BF16)
    good = make_adapter(gen, k, n, 40, BF16)
    bad = [t.clone() for t in make_adapter(gen, k, n, 20, BF16)]
    bad[0][3, 5] = float("nan")
    bad[1][:, 2] = float("inf")
    s.load(0, *bad, 1.0)
    s.load(2, *good, 0.5)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    sl = np.where(np.arange(rows) < rows // 2, np.arange(rows) % 2 * 2, np.arange(rows) // 20 % 2 * 2).astype(np.int32)
    xd, sd = torch.from_numpy(x).to(DEV), torch.from_numpy(sl).to(DEV)
    ctx = ov.default_context()
    if force:
        ctx.set_batched_kernel(force)
    try:
        base = ov.project(w, xd, rows=rows).cpu().numpy().reshape(rows, n)
        got = ov.project_adapters([w], [s], xd, sd, rows)[0].cpu().numpy().reshape(rows, n)
    finally:
        ctx.set_batched_kernel("auto")
    mine = sl == 2
    check(got[mine], base[mine], x[mine], {2: (*good, 0.5)}, sl[mine], "the good rows")
    assert not np.isfinite(got[~mine]).any()
