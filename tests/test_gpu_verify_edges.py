"""Verification of drafted tokens where probabilities leave fp64's normal range: a token is drawn wherever the row has a
distribution, and never one whose probability is zero in 64 bits.

exp(-744.44) is the smallest number of fp64, one unit of 2^-1074; the logits below are so far from a rounding's border (0.85, 2.1 and
0.42 units, thirds of a unit) that an error of 1e-11 changes no unit. Pieces: the 4096 tokens whose sums are kept together.
"""
import sys

import numpy as np
import pytest

from test_gpu_verify import run

pytestmark = pytest.mark.gpu

F = np.float32
PIECE = 4096


def one_row(vocab, at):
    row = np.full((1, vocab), -2000.0, F)
    for tokens, logit in at:
        row[0, tokens] = logit
    return row


# the least token's piece among the first 64, which a wave holds, and behind them
@pytest.mark.parametrize("first,vocab", [(0, 3 * PIECE), (2, 3 * PIECE), (66, 70 * PIECE + 5)])
@pytest.mark.parametrize("tokens", [2, 4, 40])
def test_a_piece_whose_tokens_all_round_to_zero(first, vocab, tokens):
    # one unit each before the division by the row's sum of 3, none after it; their sum alone would be left
    print("[case]", first, vocab, tokens, flush=True, file=sys.stderr)
    low = first * PIECE + 7 + np.arange(tokens)
    row = one_row(vocab, [(low, -744.6), (vocab - 1 - np.arange(3), 0.0)])
    off, none = np.array([0, 1], np.int32), np.zeros(0, np.int32)
    for last in (0.0, 0.4, 1.0, 2.0):
        _, out = run(row, off, none, np.zeros(0, F), np.array([last], F))
        assert out[0] >= vocab - 3
    # behind all others: what a number past the end is given to
    high = np.concatenate([row[:, ::-1], row], 1)
    run(np.ascontiguousarray(high), off, none, np.zeros(0, F), np.array([1.0], F))


@pytest.mark.parametrize("first,vocab", [(0, 3 * PIECE), (66, 70 * PIECE + 5)])
@pytest.mark.parametrize("probs", [False, True])
def test_a_refused_draft_alone_in_its_piece(first, vocab, probs):
    # the draft has two units; the others of its piece add up to two with it, but round to zero each
    print("[case]", first, vocab, probs, flush=True, file=sys.stderr)
    x = first * PIECE + 9
    row = one_row(vocab, [([x], -743.7), (x + 1 + np.arange(5), -745.3), ([vocab - 1], 0.0)])
    logits, off = np.concatenate([row, row]), np.array([0, 2], np.int32)
    q = None
    if probs:
        q = np.zeros((1, vocab), F)
        q[0, x] = 1.0
    for last in (0.0, 0.5, 1.0):
        accepted, out = run(logits, off, np.array([x], np.int32), np.array([0.5], F), np.array([last], F), q)
        assert accepted[0] == 0 and out[0] == vocab - 1


@pytest.mark.parametrize("temperature", [1.0, 0.01, 3.0])
def test_units_are_weights(temperature):
    # tokens of a unit or more are drawn by a number of zero: the first of them
    row = one_row(9000, [([100], -743.7 * temperature), ([50], -746.0 * temperature), ([8000], 0.0)])
    row[row == -2000.0] = -2000.0 * max(1.0, temperature)
    off, none = np.array([0, 1], np.int32), np.zeros(0, np.int32)
    t = np.array([temperature], F)
    for last in (0.0, 0.5):
        run(row, off, none, np.zeros(0, F), np.array([last], F), temperature=t)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab", [2, 25, 460, 9000])
def test_a_number_of_one_gives_the_last_token_with_a_weight(vocab, probs):
    # no running sum passes the whole total, also not one that was rounded up
    print("[case]", vocab, probs, flush=True, file=sys.stderr)
    rng = np.random.default_rng(vocab)
    requests = 300 if vocab < 5000 else 60
    logits = (rng.standard_normal((2 * requests, vocab)) * rng.choice([1.0, 20.0, 150.0], (2 * requests, 1))).astype(F)
    logits[rng.random(logits.shape) < 0.2] = -np.inf
    logits[:, 0] = 1.0
    off = (2 * np.arange(requests + 1)).astype(np.int32)
    drafts = rng.integers(0, vocab, requests).astype(np.int32)
    q = None
    if probs:
        q = rng.random((requests, vocab)).astype(F) ** 8
        q /= q.sum(1, keepdims=True)
    u = rng.random(requests).astype(F)
    last = rng.choice(np.array([1.0, 1.5, np.inf, np.nan], F), requests)
    _, out = run(logits, off, drafts, u, last, q)
    assert (out.reshape(requests, 2).max(1) >= 0).all()
