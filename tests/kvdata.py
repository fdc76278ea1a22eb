"""Paged caches filled for tests, and attention over them in 64 bits.

Tolerances, u = 2^-24. A query enters the products with an error of at most 2^-23 of its row's largest channel, the products of a
score are added up in (parts * channels + 8) steps of at most 2 u of the sum of magnitudes (three parts beside bf16 keys, else two),
and a score, a difference from its reference and their powers are rounded a few times:
  ds = 2^-23 max|q| sum|k| + (3 D + 8) 2 u sum|q k| + 6 u |s| + 8 u
A weight is off by the factor exp(2 ds) at most against the others, 2^-22 for its parts, and 2^-34 of the largest weight for those
that fp16 cannot hold; the sums over n tokens take (3 n + 64) steps of 2 u.
"""
import math
import sys

import numpy as np
import torch

U = 2.0 ** -24
DEV = "cuda:0"
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": None}


def case(*what):
    print("[case]", *what, flush=True, file=sys.stderr)


def type_id(ov, name):
    return {"f16": ov.TYPE_F16, "bf16": ov.TYPE_BF16, "i8": ov.TYPE_I8}[name]


def quantised(x):
    """(quants, scales) of 8-bit caches, in the 32-bit steps that define them; x [..., channels] fp32."""
    s = np.abs(x).max(-1, keepdims=True) / np.float32(127)
    inv = np.where(s > 0, np.float32(1) / np.where(s > 0, s, np.float32(1)), np.float32(0))
    return np.clip(np.rint(x * inv), -127, 127).astype(np.float32), s


def as_stored(x, type_):
    """What a cache of the type holds for fp32 values, in 64 bits."""
    if type_ == "i8":
        q, s = quantised(x)
        return q.astype(np.float64) * s.astype(np.float64)
    return torch.from_numpy(x).to(DTYPE[type_]).double().numpy()


class Requests:
    """Requests with `contexts` tokens each in a cache and `counts` new ones: keys, values, tables, and calls with them."""

    def __init__(self, ov, rng, type_, kv_heads, dim, page, counts, contexts, sums=False, extra=2, spread=1.0):
        self.ov, self.type_, self.kv_heads, self.dim, self.page = ov, type_, kv_heads, dim, page
        self.counts, self.contexts = list(counts), list(contexts)
        self.lengths = [n + m for n, m in zip(counts, contexts)]
        need = [-(-n // page) for n in self.lengths]
        self.width = max(max(need), 1) + 1
        self.pages = sum(need) + extra
        order = rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((len(counts), self.width), -7, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.tables[r, :n] = order[at:at + n]
            at += n
        self.off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.off[-1])
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.k = [f(n, kv_heads, dim) * np.float32(spread) for n in self.lengths]
        self.v = [f(n, kv_heads, dim) + np.float32(0.3) for n in self.lengths]
        self.cache = ov.KvCache(kv_heads, dim, page, self.pages, type_id(ov, type_), sums=sums)

    def t(self, x):
        return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)

    def batch(self, device=True):
        x = (self.off, np.array(self.lengths, np.int32), self.tables)
        return tuple(self.t(v) for v in x) if device else x

    def fill(self, upto=None):
        """Appends every request's tokens in two calls, the second over all requests."""
        for r, n in enumerate(self.lengths):
            first = n // 3
            if first:
                self.ov.kv_append(self.cache, self.t(self.k[r][:first].reshape(first, -1)), self.t(self.v[r][:first].reshape(first, -1)),
                                  self.t(np.array([0, first], np.int32)), self.t(np.array([first], np.int32)), self.t(self.tables[r:r + 1]))
        rest = [n - n // 3 for n in self.lengths]
        if sum(rest):
            flat = lambda x: self.t(np.concatenate([v[len(v) // 3:] for v in x]).reshape(sum(rest), -1))  # noqa: E731
            off = np.concatenate([[0], np.cumsum(rest)]).astype(np.int32)
            self.ov.kv_append(self.cache, flat(self.k), flat(self.v), self.t(off), self.t(np.array(self.lengths, np.int32)),
                              self.t(self.tables))
        return self

    def stored(self, r):
        """Request r's (keys, values) [tokens][kv_heads][dim] as its cache holds them."""
        return as_stored(self.k[r], self.type_), as_stored(self.v[r], self.type_)


def attention(req, q, heads, scale=None, window=0, keep=None, stored=None):
    """(out, tolerance) [rows][heads * dim] in 64 bits; keep(row, kv head, tokens): which of the row's tokens count."""
    dim, hk = req.dim, req.kv_heads
    group = heads // hk
    scale = 1 / math.sqrt(dim) if scale is None else float(np.float32(scale))
    q = q.reshape(req.rows, heads, dim).astype(np.float64)
    out, err = np.zeros((req.rows, heads, dim)), np.zeros((req.rows, heads, dim))
    for r in range(len(req.counts)):
        k, v = (stored or req.stored)(r)
        for i in range(req.counts[r]):
            row, p = req.off[r] + i, req.contexts[r] + i
            first = max(0, p - window + 1) if window else 0
            for a in range(hk):
                seen = np.arange(first, p + 1)
                if keep is not None:
                    seen = seen[keep(row, a, seen)]
                if not len(seen):
                    continue
                kk, vv, qq = k[seen, a], v[seen, a], q[row, a * group:(a + 1) * group]
                s = qq @ kk.T * scale
                ds = abs(scale) * (2 ** -23 * np.abs(qq).max(1)[:, None] * np.abs(kk).sum(1) + (3 * dim + 8) * 2 * U * (np.abs(qq) @ np.abs(kk).T))
                ds = ds + 6 * U * np.abs(s) + 8 * U
                e = np.exp(s - s.max(1, keepdims=True))
                w = e / e.sum(1, keepdims=True)
                o = w @ vv
                rel = np.expm1(2 * ds.max(1)) + 2 ** -22 + 2 * (3 * len(seen) + 64) * 2 * U
                out[row, a * group:(a + 1) * group] = o
                err[row, a * group:(a + 1) * group] = (w @ np.abs(vv) + np.abs(o)) * rel[:, None] + 2 ** -34 * np.abs(vv).sum(0) + 1e-30
    return out.reshape(req.rows, -1), err.reshape(req.rows, -1)


def check(got, want, err, what="", whole=True):
    got = got.detach().cpu().numpy().reshape(want.shape) if isinstance(got, torch.Tensor) else got.reshape(want.shape)
    off = np.abs(got - want) / (err + 1e-300)
    off = np.where(np.isfinite(got), off, np.inf)
    assert np.all(off <= 1), f"{what}: {np.max(off):.2f} times the tolerance at {np.unravel_index(np.argmax(off), off.shape)}"
    # A lost part of q or p would show as 2^-12 (2^-9 for bf16): far above what the roundings above add up to on the whole, where scores
    # are of the order of 10 at most (beyond, the score's own rounding to fp32 alone comes to that).
    n = np.linalg.norm(want)
    assert not whole or n == 0 or np.linalg.norm(got - want) / n < 1e-5, f"{what}: {np.linalg.norm(got - want) / n:.2g} off on the whole"
