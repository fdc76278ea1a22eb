"""The norms around the residual sum (ovfq_residual_norm[_dev]) against the same step in 64 bits.

Tolerance, u = 2^-24: a sum over the row runs in partial sums of at most 64 terms a thread (rows up to 16384; k / 1024 above),
joined in at most 16 more, n = max(64, k / 1024) + 16 additions; so a mean of squares is (n + 2) u off, relative, its root half
of that, and a normalised element (n / 2 + 8) u with the division, the products and the bias. Layer norms subtract a mean that
is n u mean|v| off. An error e of the input shifts a normalised element by |w| r (|e| + mean|e|) and, through the root, by
|x| rms(e) / rms(v).
"""
import ctypes
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ov = pytest.importorskip("overfit_amd")
from overfit_amd import _lib  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24


def case(*what):
    print("[case]", *what, flush=True, file=sys.stderr)


def normed(v, err, n):
    """(norm of v, its error) for inputs that are `err` off."""
    k = v.shape[1]
    terms = max(64, k / 1024) + 16
    w = 1.0 if n.weight is None else n.weight.astype(np.float64)
    b = 0.0 if n.bias is None else n.bias.astype(np.float64)
    e = err
    if n.kind == "layer":
        mean_err = terms * U * np.abs(v).mean(1, keepdims=True) + err.mean(1, keepdims=True)
        v = v - v.mean(1, keepdims=True)
        e = err + mean_err + U * np.abs(v)
    ms = np.square(v).mean(1, keepdims=True) + n.eps
    r = 1 / np.sqrt(ms)
    out = v * r * w
    rel = np.sqrt(np.square(e).mean(1, keepdims=True)) * r + (terms / 2 + 8) * U
    return out + b, np.abs(w) * r * e + np.abs(out) * rel + 2 * U * np.abs(out + b)


def reference(y, h, post, gate, axis, scale, pre):
    v, err = y.astype(np.float64), np.zeros(y.shape)
    if post is not None:
        v, err = normed(v, err, post)
    g = 1.0 if gate is None else gate.astype(np.float64).reshape((-1, 1) if axis == "row" else gate.shape)
    f = np.float64(np.float32(scale)) * g
    v, err = v * f, np.abs(f) * err + 3 * U * np.abs(v * f)
    if h is not None:
        v = v + h
        err = err + U * np.abs(v)
    return (v, err) + (normed(v, err, pre) if pre is not None else (None, None))


def inputs(rng, rows, k, kind, post, gate, residual, pre):
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    norm = lambda: ov.Norm(1 + 0.3 * f(k), 0.2 * f(k) if kind == "layer" else None, 1e-5, kind)  # noqa: E731
    shape = {None: None, "channel": (k,), "row": (rows,), "full": (rows, k)}[gate]
    return (f(rows, k) + np.float32(0.5), 2 * f(rows, k) if residual else None, norm() if post else None,
            None if shape is None else f(*shape), norm() if pre else None)


def on_device(v):
    if isinstance(v, ov.Norm):
        return ov.Norm(on_device(v.weight), on_device(v.bias), v.eps, v.kind)
    return None if v is None else torch.from_numpy(np.ascontiguousarray(v)).to(DEV)


def check(got, want, err, what):
    got = got.reshape(want.shape)
    off = np.abs(got - want) / (err + 1e-300)
    assert np.all(off <= 1), f"{what}: {np.max(off):.2f} times the tolerance at {np.unravel_index(np.argmax(off), off.shape)}"


def run(rows, k, kind="rms", post=True, gate=None, residual=True, pre=True, scale=0.7, host=False):
    case(rows, k, kind, post, gate, residual, pre, scale, host)
    rng = np.random.default_rng(rows * 131 + k)
    y, h, po, g, pr = inputs(rng, rows, k, kind, post, gate, residual, pre)
    if host:
        ho, xo = ov.residual_norm(y, rows, h, po, g, gate, scale, pr)
    else:
        ho, xo = ov.residual_norm(on_device(y), rows, on_device(h), on_device(po), on_device(g), gate, scale, on_device(pr))
        ho, xo = (None if v is None else v.cpu().numpy() for v in (ho, xo))
    want = reference(y, h, po, g, gate, scale, pr)
    if ho is None:
        assert not (post or gate or residual) and pre
    else:
        check(ho, want[0], want[1], "h")
    if pre:
        check(xo, want[2], want[3], "x")
    else:
        assert xo is None


# widths on both sides of every kernel's limit, odd ones (rows that start on no 16-byte boundary), one element
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 2), (5, 3), (17, 64), (33, 65), (9, 127), (70, 128), (7, 129), (5, 255), (6, 256),
                                    (3, 257), (4, 512), (9, 513), (2, 1023), (5, 1024), (3, 1025), (2, 2048), (3, 2049),
                                    (2, 4096), (3, 4099), (2, 8192), (2, 8193), (2, 16384), (2, 16385), (3, 20001), (1, 70000)])
def test_widths(kind, rows, k):
    run(rows, k, kind)


@pytest.mark.parametrize("k", [96, 701, 4096, 17000])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "row", "full"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("pre", [False, True])
def test_parts(k, post, gate, residual, pre):
    run(5, k, "layer" if k == 701 else "rms", post, gate, residual, pre)


@pytest.mark.parametrize("rows,k", [(1, 4096), (2048, 4096), (10592, 128), (513, 5120), (300, 14336)])
def test_model_sizes(rows, k):
    run(rows, k, gate="channel")


@pytest.mark.parametrize("k", [80, 1000, 18000])
def test_host_pointers(k):
    run(6, k, "layer", gate="full", host=True)
    run(6, k, "rms", post=False, residual=False, host=True)


@pytest.mark.parametrize("k", [100, 2051, 16500])
def test_in_place(k):
    # the residual plane updated where it lies, and the normed plane over the block's output
    rng = np.random.default_rng(k)
    rows = 7
    y, h, po, g, pr = inputs(rng, rows, k, "rms", True, "full", True, True)
    yd, hd = on_device(y), on_device(h)
    ov.residual_norm(yd, rows, hd, on_device(po), on_device(g), "full", 0.5, on_device(pr), h_out=hd, x_out=yd)
    want = reference(y, h, po, g, "full", 0.5, pr)
    check(hd.cpu().numpy(), want[0], want[1], "h in place")
    check(yd.cpu().numpy(), want[2], want[3], "x over y")
    yd, hd = on_device(y), on_device(h)
    ov.step._norm_call(yd, rows, hd, on_device(po), None, None, 0.5, on_device(pr), None, hd, None, False)[0]()
    want = reference(y, h, po, None, None, 0.5, pr)
    check(hd.cpu().numpy(), want[2], want[3], "x over the residual")
    yd = on_device(y)
    ov.residual_norm(yd, rows, on_device(h), h_out=yd, scale=-2.0)
    want = reference(y, h, None, None, None, -2.0, None)
    check(yd.cpu().numpy(), want[0], want[1], "h over y")


@pytest.mark.parametrize("k", [128, 1000, 4096, 17000])
def test_rows_keep_to_themselves(k):
    # zeros, huge and tiny rows, infinities and NaN: no row changes another, and a zero row stays finite
    rng = np.random.default_rng(k)
    rows = 9
    y = rng.standard_normal((rows, k)).astype(np.float32)
    y[1] = 0
    y[3] *= np.float32(1e15)
    y[4] *= np.float32(1e-15)
    y[5, k // 2] = np.inf
    y[7, 0] = np.nan
    pr = ov.Norm(eps=1e-6)
    _, x = ov.residual_norm(on_device(y), rows, pre=pr)
    x = x.cpu().numpy().reshape(rows, k)
    good = [0, 1, 2, 3, 4, 6, 8]
    want = reference(y[good], None, None, None, None, 1.0, pr)
    check(x[good], want[2], want[3] + 1e-38, "the finite rows")
    assert not x[1].any()
    assert np.isnan(x[7]).all() and not np.isfinite(x[5]).all()


@pytest.mark.parametrize("k", [64, 1500])
def test_layer_norm_of_a_large_offset(k):
    # mean 1e4 over deviations of 1: the squares are taken of the deviations
    rng = np.random.default_rng(k)
    y = (rng.standard_normal((4, k)) + 1e4).astype(np.float32)
    pr = ov.Norm(kind="layer")
    _, x = ov.residual_norm(on_device(y), 4, pre=pr)
    want = reference(y, None, None, None, None, 1.0, pr)
    check(x.cpu().numpy(), want[2], want[3], "x")


@pytest.mark.parametrize("k", [130, 3001])
def test_planes_on_any_4_byte_boundary(k):
    rng = np.random.default_rng(k)
    rows = 5
    y, h, _, g, pr = inputs(rng, rows, k, "rms", False, "full", True, True)
    want = reference(y, h, None, g, "full", 1.0, pr)

    def shifted(v, by):
        t = torch.full((v.size + 8,), 77.0, device=DEV)
        t[by:by + v.size] = torch.from_numpy(v.reshape(-1))
        return t, t[by:by + v.size]

    planes = [shifted(v, by) for v, by in ((y, 1), (h, 2), (g, 3), (np.zeros_like(y), 1), (np.zeros_like(y), 3))]
    (_, yd), (_, hd), (_, gd), (hw, ho), (xw, xo) = planes
    ov.residual_norm(yd, rows, hd, None, gd, "full", 1.0, ov.Norm(on_device(pr.weight)), h_out=ho, x_out=xo)
    check(ho.cpu().numpy(), want[0], want[1], "h")
    check(xo.cpu().numpy(), want[2], want[3], "x")
    for whole, by in ((hw, 1), (xw, 3)):  # nothing written outside the planes
        edge = torch.cat([whole[:by], whole[by + rows * k:]])
        assert (edge == 77.0).all()


def test_captured_call():
    rng = np.random.default_rng(2)
    rows, k = 6, 1000
    y, h, po, g, pr = inputs(rng, rows, k, "rms", True, "row", True, True)
    dev = [on_device(v) for v in (y, h, po, g, pr)]
    ho, xo = torch.empty(rows, k, device=DEV), torch.empty(rows, k, device=DEV)
    ctx = ov.default_context()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        call = ctx.bind_residual_norm_dev(dev[0], rows, dev[1], dev[2], dev[3], "row", 0.3, dev[4], ho, xo)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for step in range(3):
            dev[0].copy_(torch.from_numpy(y * (step + 1)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = reference(y * np.float32(step + 1), h, po, g, "row", 0.3, pr)
            check(ho.cpu().numpy(), want[0], want[1], f"h, replay {step}")
            check(xo.cpu().numpy(), want[2], want[3], f"x, replay {step}")
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


def test_c_entry_refusals():
    lib = _lib.load()
    ctx = ov.default_context()
    t = torch.zeros(4096, device=DEV)
    p = t.data_ptr()
    norm = lambda kind=0, eps=1e-5, w=None: ctypes.byref(_lib.NormStruct(kind, eps, w, None))  # noqa: E731

    def call(y=p, h=None, rows=2, k=64, post=None, gate=None, mode=0, pre=None, ho=p + 2048, xo=None):
        return lib.ovfq_residual_norm_dev(ctx.handle, y, h, rows, k, post, gate, mode, 1.0, pre, ho, xo)

    assert call() == 0
    for kw, want in [(dict(y=None), _lib.OVFQ_ERR_NULL), (dict(rows=0), _lib.OVFQ_ERR_RANGE), (dict(k=0), _lib.OVFQ_ERR_RANGE),
                     (dict(rows=1 << 20, k=1 << 11), _lib.OVFQ_ERR_SIZE), (dict(post=norm(2)), _lib.OVFQ_ERR_RANGE),
                     (dict(post=norm(0, -1.0)), _lib.OVFQ_ERR_RANGE), (dict(post=norm(0, float("nan"))), _lib.OVFQ_ERR_RANGE),
                     (dict(post=norm(0, 1e-5, p + 1)), _lib.OVFQ_ERR_SIZE), (dict(mode=4), _lib.OVFQ_ERR_RANGE),
                     (dict(mode=1), _lib.OVFQ_ERR_NULL), (dict(gate=p), _lib.OVFQ_ERR_NULL), (dict(ho=None), _lib.OVFQ_ERR_NULL),
                     (dict(pre=norm()), _lib.OVFQ_ERR_NULL), (dict(xo=p + 4096), _lib.OVFQ_ERR_NULL),
                     (dict(pre=norm(), xo=p + 2048), _lib.OVFQ_ERR_SIZE), (dict(y=p + 2), _lib.OVFQ_ERR_SIZE),
                     (dict(pre=norm(), h=p + 4096, xo=p + 4096), _lib.OVFQ_ERR_SIZE)]:
        assert call(**kw) == want, kw
