"""Verification of drafted tokens (ovfq_verify_drafts[_dev]) against the rule written out request by request in 64 bits.

Both sides keep probabilities and running sums in fp64 (the library's exponentials are within 2.5e-12 of their values), so counts
and tokens are equal unless a given random number falls within about 1e-11 of a border: none of the inputs here is made to.
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
F = np.float32


def case(*what):
    print("[case]", *what, flush=True, file=sys.stderr)


def target(logits, temperature):
    """The target's distribution of one row, or None without a finite largest logit."""
    v = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    m = v.max()
    if not np.isfinite(m):
        return None
    if not (0 < temperature < np.inf):
        p = np.zeros(len(v))
        p[int(np.argmax(v == m))] = 1
        return p
    e = np.exp((v - m) / np.float64(temperature))
    return e / e.sum()


def reference(logits, off, tokens, u, last, q=None, temperature=None):
    accepted, out = [], []
    for r in range(len(off) - 1):
        n, mine, w = off[r + 1] - off[r] - 1, [], None
        for i in range(n + 1):
            p = target(logits[off[r] + i], 1.0 if temperature is None else temperature[r])
            w = p
            if i == n:
                break
            d = off[r] - r + i
            x = int(tokens[d])
            qr = None
            if q is not None:
                qr = np.where(q[d] > 0, q[d].astype(np.float64), 0.0)
            inside = 0 <= x < logits.shape[1]
            if p is not None and inside and np.float64(u[d]) * (1.0 if qr is None else qr[x]) < p[x]:
                mine.append(x)
                continue
            if p is not None:
                if qr is None:
                    rest = p.copy()
                    if inside:
                        rest[x] = 0
                else:
                    rest = np.maximum(p - qr, 0)
                if rest.sum() > 0:
                    w = rest
            break
        if w is None:
            final = -1
        else:
            run = np.cumsum(w)
            over = np.flatnonzero(run > np.float64(last[r]) * run[-1])
            final = int(over[0]) if len(over) else int(np.flatnonzero(w)[-1])
        accepted.append(len(mine))
        out += mine + [final] + [-1] * (n - len(mine))
    return np.array(accepted, np.int32), np.array(out, np.int32)


def make(rng, counts, vocab, probs, masked=0.0):
    off = np.concatenate([[0], np.cumsum(np.array(counts) + 1)]).astype(np.int32)
    rows, drafts = int(off[-1]), sum(counts)
    logits = (rng.standard_normal((rows, vocab)) * 2).astype(F)
    logits[np.arange(rows), rng.integers(0, vocab, rows)] += F(9)
    if masked:
        logits[:, rng.random(vocab) < masked] = -np.inf
        logits[:, vocab // 2] = 0.5  # one token at least stays
    tokens = np.zeros(drafts, np.int32)
    q = None
    if drafts:
        rows_of = np.concatenate([off[r] + np.arange(c) for r, c in enumerate(counts)]).astype(int)
        near = np.where(np.isfinite(logits[rows_of]), logits[rows_of], -5).astype(np.float64)
        near += 0.5 * rng.standard_normal(near.shape)
        e = np.exp(near - near.max(1, keepdims=True))
        q = (e / e.sum(1, keepdims=True)).astype(F)
        run = np.cumsum(q.astype(np.float64), 1)
        tokens = (run < rng.random((drafts, 1)) * run[:, -1:]).sum(1).astype(np.int32)
    return logits, off, tokens, rng.random(drafts).astype(F), rng.random(len(counts)).astype(F), q if probs else None


def dev(v):
    return None if v is None else torch.from_numpy(np.ascontiguousarray(v)).to(DEV)


def run(logits, off, tokens, u, last, q=None, temperature=None, host=False):
    args = (logits, off, tokens, u, last, q, temperature)
    lg, of, tk, uu, la, qq, te = args if host else [dev(v) for v in args]
    got = ov.verify_drafts(lg, logits.shape[1], of, tk, uu, la, qq, te)
    got = got if host else [g.cpu().numpy() for g in got]
    want = reference(*args)
    assert np.array_equal(got[0], want[0]), (got[0], want[0])
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    return got


# vocabularies on both sides of a piece (8192 tokens), of a four-token load and of one token; requests without drafts
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("counts,vocab", [
    ((0,), 1), ((1,), 1), ((3,), 2), ((2, 0, 1), 5), ((4, 4), 257), ((1, 0, 7, 3), 1000), ((0, 0, 0), 4096), ((5, 2), 8191),
    ((2,), 8192), ((3, 1, 0), 8193), ((4, 6, 1, 0, 2), 32001), ((7, 7), 40960), ((20, 1), 9001), ((300,), 33),
])
def test_matches_the_rule(counts, vocab, probs):
    case(counts, vocab, probs)
    rng = np.random.default_rng(vocab + sum(counts))
    for _ in range(3):
        run(*make(rng, counts, vocab, probs))


@pytest.mark.parametrize("probs", [False, True])
def test_model_sizes(probs):
    rng = np.random.default_rng(7)
    counts = [7 - r % 8 for r in range(16)]
    kept = 0
    temperature = (0.3 + rng.random(16)).astype(F)
    data = make(rng, counts, 128256, probs)
    kept = run(*data, temperature=temperature)[0].sum()
    assert 0 < kept < sum(counts)  # some drafts accepted, some refused


@pytest.mark.parametrize("probs", [False, True])
def test_temperatures(probs):
    # each request its own; 0, negative, NaN and infinite ones are greedy
    rng = np.random.default_rng(11)
    temperature = np.array([1.0, 0.0, 0.05, -1.0, np.nan, 30.0, np.inf, 1e-30, 0.7], F)
    for _ in range(4):
        run(*make(rng, [3] * 9, 9000, probs), temperature=temperature)


def test_greedy_ties_take_the_first():
    logits = np.zeros((3, 20000), F)
    logits[0, [9000, 15000, 300]] = 5
    logits[1, [8191, 8192]] = 2
    off, zero = np.array([0, 3], np.int32), np.zeros(1, F)
    got = run(logits, off, np.array([300, 8191], np.int32), np.array([0.9, 0.9], F), np.array([0.5], F), None, zero)
    assert got[0][0] == 2 and list(got[1]) == [300, 8191, 0]


@pytest.mark.parametrize("probs", [False, True])
def test_masked_vocabulary(probs):
    rng = np.random.default_rng(5)
    for _ in range(3):
        data = make(rng, [4, 0, 5, 2], 17000, probs, masked=0.97)
        _, tokens = run(*data)
        picked = tokens[tokens >= 0]
        assert np.isfinite(data[0][:, picked]).any(0).all()


@pytest.mark.parametrize("probs", [False, True])
def test_rows_without_a_distribution(probs):
    # all -inf, all NaN, +inf: the draft is refused and nothing is drawn; NaN among others is no token
    rng = np.random.default_rng(6)
    logits, off, tokens, u, last, q = make(rng, [2, 2, 2, 2, 2], 8300, probs)
    logits[off[0]] = -np.inf
    logits[off[1] + 1] = np.nan
    logits[off[2], 8299] = np.inf
    logits[off[3] + 2] = -np.inf
    logits[off[4], ::2] = np.nan
    u[:] = 0  # every draft with a probability is kept
    accepted, out = run(logits, off, tokens, u, last, q)
    assert accepted[0] == 0 and out[off[0]] == -1
    run(logits, off, tokens, u, last, q, np.zeros(5, F))


def test_lowest_values_as_masks():
    # a mask of the type's lowest value, not an infinity
    rng = np.random.default_rng(8)
    logits, off, tokens, u, last, q = make(rng, [3, 3], 9000, True)
    logits[:, 100:] = np.finfo(F).min
    tokens %= 100
    run(logits, off, tokens, u, last, q)
    run(np.full_like(logits, np.finfo(F).min), off, tokens, u, last, q)


def test_draft_probabilities_at_their_edges():
    # a drafter that is as sure as the target, surer, contradicts itself, or gives zeros, negatives or NaN
    rng = np.random.default_rng(9)
    vocab = 500
    logits, off, tokens, u, last, _ = make(rng, [1] * 8, vocab, True)
    q = np.stack([target(logits[off[r]], 1.0) for r in range(8)]).astype(F)
    q[1] = 1.0                        # above p everywhere: nothing left beside it
    u[1] = 0.99999
    q[2] = 0.0
    q[3] = np.nan
    q[4] = -1.0
    q[5, tokens[5]] = 0.0             # says it could not have drafted that
    q[6] = 0.0
    q[6, 7] = np.inf
    u[6], tokens[6] = 0.5, 7
    run(logits, off, tokens, u, last, q)


@pytest.mark.parametrize("probs", [False, True])
def test_random_numbers_at_their_ends(probs):
    rng = np.random.default_rng(10)
    logits, off, tokens, u, last, q = make(rng, [3, 3, 3, 3], 8500, probs)
    below_one = np.nextafter(F(1), F(0))
    u[:] = [0, 0, 0, below_one, below_one, below_one, 0, 0, 0, 1, 1, 1]
    last[:] = [0, below_one, 1, 2]
    run(logits, off, tokens, u, last, q)


def test_drafts_outside_the_vocabulary():
    rng = np.random.default_rng(13)
    logits, off, tokens, u, last, q = make(rng, [3, 3, 3], 300, False)
    u[:] = 0
    tokens[1], tokens[3], tokens[8] = 300, -1, 2 ** 31 - 1
    accepted, _ = run(logits, off, tokens, u, last, None)
    assert list(accepted) == [1, 0, 2]


@pytest.mark.parametrize("probs", [False, True])
def test_host_pointers(probs):
    rng = np.random.default_rng(14)
    run(*make(rng, [2, 0, 3], 8200, probs), temperature=np.array([1, 0, 0.5], F), host=True)
    run(*make(rng, [0, 0], 100, probs), host=True)


def test_bad_offsets_on_the_device():
    # a request whose offsets do not grow or leave the rows is refused alone; its rows stay as they were
    rng = np.random.default_rng(15)
    logits, off, tokens, u, last, q = make(rng, [2, 2, 2, 2], 900, True)
    good = reference(logits, off, tokens, u, last, q)
    for bad in ([0, 3, 3, 9, 12], [0, 3, 6, 9, 13], [0, 3, 6, 9, 2 ** 31 - 1], [-3, 3, 6, 9, 12], [0, 3, 6, 5, 12]):
        bad = np.array(bad, np.int32)
        acc, tok = torch.full((4,), 99, dtype=torch.int32, device=DEV), torch.full((12,), 99, dtype=torch.int32, device=DEV)
        ov.verify_drafts(dev(logits), 900, dev(bad), dev(tokens), dev(u), dev(last), dev(q), None, acc, tok)
        acc, tok = acc.cpu().numpy(), tok.cpu().numpy()
        for r in range(4):
            if bad[r] == off[r] and bad[r + 1] == off[r + 1]:
                assert acc[r] == good[0][r]
                assert np.array_equal(tok[off[r]:off[r + 1]], good[1][off[r]:off[r + 1]])
            elif not 0 <= bad[r] < bad[r + 1] <= 12:
                assert acc[r] == -1


def test_rows_behind_the_last_request_stay():
    rng = np.random.default_rng(16)
    logits, off, tokens, u, last, q = make(rng, [2, 3, 1], 700, False)
    want = reference(logits[:7], off[:3], tokens, u, last)
    acc, tok = torch.full((2,), 99, dtype=torch.int32, device=DEV), torch.full((9,), 99, dtype=torch.int32, device=DEV)
    few = dev(np.concatenate([tokens, np.zeros(4, np.int32)]))
    uu = dev(np.concatenate([u, np.zeros(4, F)]))
    ov.verify_drafts(dev(logits), 700, dev(off[:3]), few, uu, dev(last), None, None, acc, tok)
    assert np.array_equal(acc.cpu().numpy(), want[0])
    assert np.array_equal(tok.cpu().numpy()[:7], want[1]) and (tok[7:] == 99).all()


# on both sides of a wave's 2048 logits and of the 64 pieces of 4096 tokens that a wave holds
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("counts,vocab", [((2, 1), 2047), ((2, 1), 2048), ((1, 3), 2049), ((2,), 4097), ((1, 2), 262144), ((2, 1), 262145),
                                          ((1,), 400003)])
def test_pieces(counts, vocab, probs):
    case("pieces", counts, vocab, probs)
    rng = np.random.default_rng(vocab)
    for seed in range(3):
        logits, off, tokens, u, last, q = make(rng, counts, vocab, probs)
        u = F(1) - (F(1) - u) * F(0.3) * F(seed)  # some accepted, some refused; then none accepted
        run(logits, off, tokens, np.minimum(u, np.nextafter(F(1), F(0))), last, q, rng.uniform(0.3, 2.0, len(counts)).astype(F))


@pytest.mark.parametrize("lead", [8, 14, 20, 36])
@pytest.mark.parametrize("vocab", [100, 9001])
def test_a_refused_draft_that_had_nearly_everything(vocab, lead):
    # what is left of its piece is smaller than the rounding of the piece's sum: it is summed without the draft
    case("nearly everything", vocab, lead)
    rng = np.random.default_rng(lead + vocab)
    logits = rng.standard_normal((6, vocab)).astype(F)
    at = rng.integers(0, vocab, 3)
    for r in range(3):
        logits[2 * r, at[r]] = F(lead)
    off = np.array([0, 2, 4, 6], np.int32)
    u = np.full(3, 1.0, F)  # refuses any draft
    for last in (0.0, 0.35, 0.8, 0.99999):
        run(logits, off, at.astype(np.int32), u, np.full(3, last, F))


def test_logits_far_apart():
    # beyond the smallest number's exponential: no weight, as in the 64-bit rule
    case("far apart")
    vocab = 5000
    logits = np.full((4, vocab), -760.0, F)
    logits[:, 4000] = 1.0
    logits[1, 4100] = 0.5
    logits[2, :] = np.float32(-3e38)
    logits[2, 7] = np.float32(3e38)
    logits[3, 4500] = -705.0
    off = np.arange(5, dtype=np.int32)
    none = np.zeros(0, np.int32)
    for last in (0.0, 0.5, 0.999999):
        run(logits, off, none, np.zeros(0, F), np.full(4, last, F))
        run(logits, off, none, np.zeros(0, F), np.full(4, last, F), temperature=np.array([1.0, 0.01, 1e30, 5.0], F))


def test_captured_call():
    rng = np.random.default_rng(17)
    counts = [3, 0, 4]
    data = make(rng, counts, 20000, True)
    bufs = [dev(v) for v in data]
    acc, tok = torch.empty(3, dtype=torch.int32, device=DEV), torch.empty(10, dtype=torch.int32, device=DEV)
    ctx = ov.default_context()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        call = ctx.bind_verify_drafts_dev(bufs[0], 20000, bufs[1], bufs[2], bufs[3], bufs[4], bufs[5], None, acc, tok)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(4):
            data = make(rng, counts, 20000, True)
            for b, v in zip(bufs, data):
                b.copy_(torch.from_numpy(v))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = reference(*data)
            assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
            acc.zero_()
            tok.zero_()
            torch.cuda.synchronize()
            call()
            torch.cuda.synchronize()
            assert np.array_equal(tok.cpu().numpy(), want[1])
    finally:
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)


def test_c_entry_refusals():
    lib = _lib.load()
    ctx = ov.default_context()
    f, i = torch.zeros(64, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    fp, ip = f.data_ptr(), i.data_ptr()
    i[1] = 2  # one request of two rows

    def call(logits=fp, rows=2, vocab=8, requests=1, off=ip, toks=ip + 64, q=None, u=fp, last=fp, acc=ip + 128, out=ip + 192):
        return lib.ovfq_verify_drafts_dev(ctx.handle, logits, rows, vocab, requests, off, toks, q, None, u, last, acc, out)

    assert call() == 0
    for kw, want in [(dict(logits=None), _lib.OVFQ_ERR_NULL), (dict(off=None), _lib.OVFQ_ERR_NULL),
                     (dict(last=None), _lib.OVFQ_ERR_NULL), (dict(acc=None), _lib.OVFQ_ERR_NULL),
                     (dict(out=None), _lib.OVFQ_ERR_NULL), (dict(toks=None), _lib.OVFQ_ERR_NULL),
                     (dict(u=None), _lib.OVFQ_ERR_NULL), (dict(rows=0), _lib.OVFQ_ERR_RANGE),
                     (dict(vocab=0), _lib.OVFQ_ERR_RANGE), (dict(requests=0), _lib.OVFQ_ERR_RANGE),
                     (dict(requests=3), _lib.OVFQ_ERR_SIZE), (dict(rows=65536, vocab=1 << 15), _lib.OVFQ_ERR_SIZE),
                     (dict(logits=fp + 2), _lib.OVFQ_ERR_SIZE)]:
        assert call(**kw) == want, kw
    assert call(rows=1, toks=None, u=None) == 0  # no drafts: no draft arrays (the offsets' request leaves the rows: -1)
    torch.cuda.synchronize()
    for off in ([0, 3], [1, 2], [0, 0], [0, 2, 2]):
        with pytest.raises(ov.OverfitArgumentError):
            n = len(off) - 1
            ov.verify_drafts(np.zeros(16, F), 8, np.array(off, np.int32), np.zeros(2, np.int32), np.zeros(2, F),
                             np.zeros(n, F))
