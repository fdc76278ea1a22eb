"""What a server that runs many requests through one GGUF model does around the shared quantized projections, measured.

Kinds of case (the dict's "kind"):
  adapters  projections of one activation with each request's low-rank adapter:
            y = (bias +) W q(x) + scale_s B_s (A_s x), s the row's adapter slot
  norm      the step between two blocks: h' = h + scale * gate * post_norm(y), x = pre_norm(h')
  verify    drafted tokens checked against the LM head's logits with given random numbers

Sizes follow this repository's benchmark and tests (hidden 4096, k/v 1024, FFN 14336, vocabulary 128256, heads of 128);
drawn cases spread them from 512 to 14336 inputs, 1 to 512 rows, ranks 4 to 128, vocabularies of 4000 to 151936.
Weights are GGUF blocks as a file holds them, activations and logits fp32 in device memory; q(x) is the activation in the
8-bit blocks that the weight's format prescribes (absmax / 127, ties to even).
"""
import math

import torch

own = False

DEV = "cuda:0"
Q4K, Q6K, Q8 = "q4k", "q6k", "q8_0"
ROW_BYTES = {Q4K: 144 / 256, Q6K: 210 / 256, Q8: 1.125}  # resident bytes per weight
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------- the cases

def _adapters(name, type_, ns, k, rows, requests, slots, rank, dtype, mixed=False, bias=False):
    return {"name": name, "kind": "adapters", "type": type_, "n0": ns[0], "n1": ns[1] if len(ns) > 1 else 0,
            "n2": ns[2] if len(ns) > 2 else 0, "k": k, "rows": rows, "requests": requests, "slots": slots, "rank": rank,
            "mixed": mixed, "dtype": dtype, "bias": bias}


def _norm(name, rows, k, norm="rms", post=True, gate="none", residual=True, pre=True, scale=1.0):
    return {"name": name, "kind": "norm", "rows": rows, "k": k, "norm": norm, "post": post, "gate": gate,
            "residual": residual, "pre": pre, "scale": scale}


def _verify(name, requests, drafts, vocab, probs, ragged=True, masked=0.0, greedy=False):
    return {"name": name, "kind": "verify", "requests": requests, "drafts": drafts, "vocab": vocab, "probs": probs,
            "ragged": ragged, "masked": masked, "greedy": greedy}


def listed():
    return [
        # One token of one request through a small model's output projection with a rank-8 adapter: the shortest call.
        _adapters("adapt_1row_r8", Q4K, (2048,), 2048, 1, 1, 4, 8, "bf16"),
        # A decode step of 24 requests over 16 adapters of several ranks (and one request without): q/k/v.
        _adapters("adapt_qkv_24rows", Q4K, (4096, 1024, 1024), 4096, 24, 24, 16, 16, "f16", mixed=True),
        # A request's last token and six drafted ones through the Q6_K down projection, rank 64.
        _adapters("adapt_down_7rows_r64", Q6K, (4096,), 14336, 7, 1, 8, 64, "bf16"),
        # Prompts of three requests, 331 tokens in all, through q/k/v with biases, rank 32.
        _adapters("adapt_qkv_331rows_r32", Q4K, (4096, 1024, 1024), 4096, 331, 3, 4, 32, "bf16", bias=True),
        # A Q8_0 model's projection for 45 rows of nine requests, adapters kept in fp32.
        _adapters("adapt_q8_45rows", Q8, (4096,), 4096, 45, 9, 6, 16, "f32", mixed=True),
        # A 512-token prefill chunk of two requests through gate/up, rank 16: the largest.
        _adapters("adapt_gateup_512rows", Q4K, (14336, 14336), 4096, 512, 2, 4, 16, "f16"),
        # One token between two blocks, norms on both sides of the residual.
        _norm("norm_1row", 1, 4096),
        # A prompt of 331 tokens: the norm on the query heads alone (32 heads of 128).
        _norm("norm_heads", 331 * 32, 128, post=False, residual=False),
        # A 2048-token chunk, norms on both sides, a gate for each channel and a residual scale: the largest.
        _norm("norm_2048rows_gate", 2048, 4096, gate="channel", scale=0.22),
        # One request's four drafted tokens without draft probabilities.
        _verify("verify_1request", 1, 4, 32000, False, ragged=False),
        # 16 requests with up to seven drafted tokens each and the drafter's probabilities.
        _verify("verify_16requests", 16, 7, 128256, True),
        # 48 requests with four drafted tokens each, no probabilities, under a grammar that masks half the vocabulary.
        _verify("verify_48requests_masked", 48, 4, 128256, False, ragged=False, masked=0.5),
    ]


def _logint(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["adapters", "adapters", "norm", "verify"])
    if kind == "adapters":
        type_ = rng.choice([Q4K, Q4K, Q6K, Q8])
        k = _logint(rng, 512, 14336, 32 if type_ == Q8 else 256)
        ns = [_logint(rng, 256, 14336)]
        if rng.random() < 0.5:
            ns += [max(64, ns[0] // rng.choice([1, 4, 8]))] * rng.choice([1, 2])
        rows = 1 if rng.random() < 0.2 else _logint(rng, 2, 512)
        while rows * sum(ns) * k > 6e10:  # no longer than the largest listed call
            rows //= 2
        requests = rows if rng.random() < 0.4 else _logint(rng, 1, rows)
        c = _adapters("", type_, ns, k, rows, requests, _logint(rng, 1, 32), _logint(rng, 4, 128),
                      rng.choice(["f32", "f16", "bf16"]), mixed=rng.random() < 0.5, bias=rng.random() < 0.3)
    elif kind == "norm":
        k = _logint(rng, 64, 16384)
        c = _norm("", _logint(rng, 1, max(1, min(16384, 2048 * 4096 // k))), k, norm=rng.choice(["rms", "rms", "layer"]),
                  post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "row", "full"]),
                  residual=rng.random() < 0.8, pre=rng.random() < 0.8, scale=round(rng.uniform(0.1, 1.5), 3))
    else:
        drafts = rng.randint(1, 8)
        vocab = _logint(rng, 4000, 151936)
        c = _verify("", max(1, _logint(rng, 1, 48) * 4 // (drafts + 1)), drafts, vocab, rng.random() < 0.5,
                    ragged=rng.random() < 0.7, masked=rng.choice([0.0, 0.0, 0.5, 0.95]), greedy=rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------- what it holds

def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + part)


def _u8(gen, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=gen, device=DEV, dtype=torch.uint8)


def _half_bytes(gen, nb, lo, hi):
    d = torch.rand(nb, 1, generator=gen, device=DEV) * (hi - lo) + lo
    return d.to(torch.float16).view(torch.uint8)  # [nb, 2]


def _blocks(gen, type_, n, k):
    """Weights of deviation about 0.02 as a GGUF file stores them: uint8 blocks, or (int8 quants, f32 scales) planes for
    Q8_0."""
    if type_ == Q8:
        q = (_u8(gen, 0, 128, (n * k,)).to(torch.int16) + _u8(gen, 0, 128, (n * k,)) - 127).to(torch.int8)
        s = (torch.rand(n * k // 32, generator=gen, device=DEV) * 3e-4 + 2.5e-4).to(torch.float16).float()
        return q, s
    nb = n * k // 256
    if type_ == Q4K:
        d, dmin = _half_bytes(gen, nb, 1.0e-4, 1.6e-4), _half_bytes(gen, nb, 0.9e-3, 1.2e-3)
        sc, m = _u8(gen, 24, 64, (nb, 8)), _u8(gen, 24, 64, (nb, 8))
        packed = torch.cat([sc[:, :4] | ((sc[:, 4:] >> 4) << 6), m[:, :4] | ((m[:, 4:] >> 4) << 6),
                            (sc[:, 4:] & 15) | ((m[:, 4:] & 15) << 4)], 1)
        nib = _u8(gen, 0, 8, (2, nb, 128)) + _u8(gen, 0, 9, (2, nb, 128))
        return torch.cat([d, dmin, packed, nib[0] | (nib[1] << 4)], 1).reshape(-1)
    ql = _u8(gen, 0, 256, (nb, 128))
    qh = _u8(gen, 0, 256, (nb, 64))
    sc = _u8(gen, 40, 128, (nb, 16)).to(torch.int8) * (1 - 2 * _u8(gen, 0, 2, (nb, 16)).to(torch.int8))
    return torch.cat([ql, qh, sc.view(torch.uint8), _half_bytes(gen, nb, 0.6e-5, 2.0e-5)], 1).reshape(-1)


def _ns(c):
    return [n for n in (c["n0"], c["n1"], c["n2"]) if n]


def _split(gen, total, parts):
    """`total` rows over `parts` requests of uneven lengths, at least one each: each row's request."""
    cuts = torch.randperm(total - 1, generator=gen, device=DEV)[:parts - 1] + 1 if total > 1 else torch.zeros(
        0, dtype=torch.int64, device=DEV)
    first = torch.zeros(total, dtype=torch.int64, device=DEV)
    first[cuts] = 1
    return first.cumsum(0)


def _ranks(c):
    """Each slot's rank: all the same, or falling by a quarter of it from slot to slot (at least 1)."""
    return [max(1, c["rank"] - c["rank"] * (s % 4) // 4) if c["mixed"] else c["rank"] for s in range(c["slots"])]


def _adapter_inputs(c, seed):
    gen = _gen(seed, 7)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    t, k, slots, dt = {}, c["k"], c["slots"], DTYPE[c["dtype"]]
    t["x"] = randn(c["rows"], k)
    t["bias"] = [randn(n) * 0.1 for n in _ns(c)] if c["bias"] else None
    t["blocks"] = [_blocks(_gen(seed, 100 + i), c["type"], n, k) for i, n in enumerate(_ns(c))]
    # request r has adapter r modulo (slots + 1), in a shuffled order; the last of them is "none"
    order = torch.cat([torch.randperm(slots, generator=gen, device=DEV), torch.tensor([-1], device=DEV)])
    t["slot"] = order[_split(gen, c["rows"], c["requests"]) % (slots + 1)].to(torch.int32)
    ranks = torch.tensor(_ranks(c), device=DEV)
    live = (torch.arange(c["rank"], device=DEV) < ranks[:, None])  # past a slot's rank: zeros
    t["a"] = [(randn(slots, c["rank"], k) / math.sqrt(k) * live[:, :, None]).to(dt) for _ in _ns(c)]
    t["b"] = [(randn(slots, n, c["rank"]) * 0.05 * live[:, None, :]).to(dt) for n in _ns(c)]
    t["scale"] = torch.rand(slots, generator=gen, device=DEV) * 1.5 + 0.5  # alpha / rank
    return t


def _has_sum(c):
    """Whether h' is another plane than the input (else the step is the norm alone)."""
    return c["residual"] or c["post"] or c["gate"] != "none" or not c["pre"]


def _norm_inputs(c, seed):
    gen = _gen(seed, 8)
    rows, k = c["rows"], c["k"]
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    t = {"y": randn(rows, k) * 0.7 + 0.1, "h": randn(rows, k) * 2 if c["residual"] else None}
    for name in ("post", "pre"):
        t[name] = (1 + 0.2 * randn(k), 0.1 * randn(k) if c["norm"] == "layer" else None) if c[name] else None
    shape = {"none": None, "channel": (k,), "row": (rows,), "full": (rows, k)}[c["gate"]]
    t["gate"] = None if shape is None else torch.sigmoid(randn(*shape))
    return t


def _draft_counts(c):
    return [c["drafts"] - (r % (c["drafts"] + 1) if c["ragged"] else 0) for r in range(c["requests"])]


def _verify_inputs(c, seed):
    gen = _gen(seed, 9)
    vocab = c["vocab"]
    rand = lambda *s: torch.rand(*s, generator=gen, device=DEV)  # noqa: E731
    counts = torch.tensor(_draft_counts(c), device=DEV)[torch.randperm(c["requests"], generator=gen, device=DEV)]
    off = torch.zeros(c["requests"] + 1, dtype=torch.int64, device=DEV)
    off[1:] = (counts + 1).cumsum(0)
    rows = sum(_draft_counts(c)) + c["requests"]
    logits = torch.randn(rows, vocab, generator=gen, device=DEV) * 2.5
    peaks = torch.randint(0, vocab, (rows, 8), generator=gen, device=DEV)
    logits.scatter_add_(1, peaks, 6 + 8 * rand(rows, 8))  # a model is sure of a few tokens
    if c["masked"]:
        logits[:, rand(vocab) < c["masked"]] = -math.inf
    request = torch.repeat_interleave(torch.arange(c["requests"], device=DEV), counts + 1, output_size=rows)
    is_draft = torch.arange(rows, device=DEV) - off[request] < counts[request]
    at = is_draft.nonzero().squeeze(1)  # the row that verifies each draft
    # the drafter: a small model, near the target; it drafts from its own distribution, over every token
    near = torch.where(torch.isfinite(logits[at]), logits[at], torch.full_like(logits[at], -6.0))
    q = torch.softmax(near + 0.7 * torch.randn(near.shape, generator=gen, device=DEV), 1)
    tokens = torch.multinomial(q, 1, generator=gen).squeeze(1) if len(at) else at
    temp = rand(c["requests"]) * 0.9 + 0.4
    if c["greedy"]:
        temp[::2] = 0.0  # every second request decodes greedily
    return {"logits": logits, "off": off.to(torch.int32), "tokens": tokens.to(torch.int32), "q": q if c["probs"] else None,
            "u": rand(len(at)), "last": rand(c["requests"]), "temp": temp}


def prepare(case, seed):
    st = dict(case)
    if case["kind"] == "adapters":
        st.update(_adapter_inputs(case, seed))
    elif case["kind"] == "norm":
        st.update(_norm_inputs(case, seed), axis=None if case["gate"] == "none" else case["gate"], sum=_has_sum(case))
    else:
        st.update(_verify_inputs(case, seed))
    if own:
        _prepare_own(st)
    return st


def _prepare_own(st):
    """What a server keeps: resident weights, the adapters loaded into their slots, outputs and prepared calls."""
    import overfit_amd as ov

    ctx = ov.default_context()
    new = lambda n, t=torch.float32: torch.empty(n, dtype=t, device=DEV)  # noqa: E731
    if st["kind"] == "adapters":
        cls = {Q4K: ov.Q4KWeight, Q6K: ov.Q6KWeight}
        k, ns = st["k"], _ns(st)
        if st["type"] == Q8:
            st["w"] = [ov.Q8Weight(b[0], b[1], k, n) for b, n in zip(st["blocks"], ns)]
        else:
            st["w"] = [cls[st["type"]](b, k, n) for b, n in zip(st["blocks"], ns)]
        type_ = {"f32": ov.TYPE_F32, "f16": ov.TYPE_F16, "bf16": ov.TYPE_BF16}[st["dtype"]]
        st["sets"] = [ov.AdapterSet(k, n, st["slots"], st["rank"], type_) for n in ns]
        for a, b, s in zip(st["a"], st["b"], st["sets"]):
            for slot, rank in enumerate(_ranks(st)):
                s.load(slot, a[slot, :rank], b[slot, :, :rank].contiguous(), float(st["scale"][slot]))
        st["out"] = [new(st["rows"] * n).view(st["rows"], n) for n in ns]
        st["call"] = ctx.bind_adapters_dev(st["w"], st["sets"], st["x"], st["slot"], st["out"], biases=st["bias"],
                                           rows=st["rows"])
    elif st["kind"] == "norm":
        norm = lambda p: None if p is None else ov.Norm(p[0], bias=p[1], eps=1e-5, kind=st["norm"])  # noqa: E731
        h = torch.empty_like(st["y"]) if st["sum"] else None
        st["out"] = [h, torch.empty_like(st["y"]) if st["pre"] else None]
        st["call"] = ctx.bind_residual_norm_dev(
            st["y"], st["rows"], residual=st["h"], post=norm(st["post"]), gate=st["gate"],
            gate_axis=st["axis"], scale=st["scale"], pre=norm(st["pre"]), h_out=h, x_out=st["out"][1])
    else:
        rows = st["logits"].shape[0]
        st["out"] = [new(st["requests"], torch.int32), new(rows, torch.int32)]
        st["call"] = ctx.bind_verify_drafts_dev(st["logits"], st["vocab"], st["off"], st["tokens"], st["u"], st["last"],
                                                draft_probs=st["q"], temperature=st["temp"], accepted=st["out"][0],
                                                tokens=st["out"][1])


def run(st):
    if own:
        st["call"]()
        return st["out"]
    return {"adapters": _plain_adapters, "norm": _plain_norm, "verify": _plain_verify}[st["kind"]](st)


# --------------------------------------------------------------------------------------------------- plain forms

def _weight32(type_, blocks, n, k):
    """[n][k] weights in 32 bits from their blocks."""
    if type_ == Q8:
        return (blocks[0].view(n, k // 32, 32).float() * blocks[1].view(n, k // 32, 1)).view(n, k)
    b = blocks.view(n * k // 256, -1)
    half = lambda v: v.contiguous().view(torch.float16).float()  # noqa: E731
    if type_ == Q4K:
        s = b[:, 4:16]
        sc = torch.cat([s[:, :4] & 63, (s[:, 8:] & 15) | ((s[:, :4] >> 6) << 4)], 1).float() * half(b[:, 0:2])
        m = torch.cat([s[:, 4:8] & 63, (s[:, 8:] >> 4) | ((s[:, 4:8] >> 6) << 4)], 1).float() * half(b[:, 2:4])
        qs = b[:, 16:].view(-1, 4, 1, 32)
        nib = torch.cat([qs & 15, qs >> 4], 2).view(-1, 8, 32)
        return (nib.float() * sc[:, :, None] - m[:, :, None]).view(n, k)
    ql, qh = b[:, :128].view(-1, 2, 2, 32), b[:, 128:192].view(-1, 2, 1, 32)
    q = torch.cat([ql & 15, ql >> 4], 2) | torch.cat([((qh >> s) & 3) << 4 for s in (0, 2, 4, 6)], 2)
    sc = b[:, 192:208].contiguous().view(torch.int8).float() * half(b[:, 208:210])
    return ((q.view(-1, 16, 16).float() - 32) * sc[:, :, None]).view(n, k)


def _q8(x, block):
    """q(x): blocks of `block` values as int8 times absmax / 127, in 32 bits (division by a tensor is correctly rounded)."""
    v = x.view(-1, block)
    s = v.abs().amax(1, keepdim=True)
    s = s / torch.full_like(s, 127.0)
    inv = torch.where(s > 0, torch.ones_like(s) / s, torch.zeros_like(s))
    return (torch.round(v * inv).clamp(-127, 127) * s).view(x.shape)


def _plain_adapters(st):
    x, slots, rank = st["x"], st["slots"], st["rank"]
    xq = _q8(x, 32 if st["type"] == Q8 else 256)
    mine = (st["slot"][:, None] == torch.arange(slots, device=DEV)).float() * st["scale"]  # [rows][slots]
    mine = mine.repeat_interleave(rank, 1)

    def one(blocks, n, a, b, bias):
        y = xq @ _weight32(st["type"], blocks, n, st["k"]).t()
        low = (x @ a.float().view(slots * rank, -1).t()) * mine
        y = y + low @ b.float().permute(1, 0, 2).reshape(n, slots * rank).t()
        return y if bias is None else y + bias

    return [one(*v) for v in zip(st["blocks"], _ns(st), st["a"], st["b"], st["bias"] or [None] * 3)]


def _plain_normed(v, p, norm):
    if norm == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5) * p[0]
    return v if p[1] is None else v + p[1]


def _plain_norm(st):
    if not st["sum"]:
        return [None, _plain_normed(st["y"] * st["scale"], st["pre"], st["norm"])]
    t = st["y"] if st["post"] is None else _plain_normed(st["y"], st["post"], st["norm"])
    if st["gate"] is not None:
        t = t * (st["gate"][:, None] if st["axis"] == "row" else st["gate"])
    h = t * st["scale"] if st["h"] is None else st["h"] + t * st["scale"]
    return [h, None if st["pre"] is None else _plain_normed(h, st["pre"], st["norm"])]


def _plain_verify(st):
    """Probabilities and their running sums in 64 bits: a draw falls between two of them."""
    off, rows = st["off"].long(), st["logits"].shape[0]
    requests, drafts = st["requests"], st["tokens"].long()
    request = torch.repeat_interleave(torch.arange(requests, device=DEV), off[1:] - off[:-1], output_size=rows)
    count = (off[1:] - off[:-1] - 1)[request]
    place = torch.arange(rows, device=DEV) - off[request]
    temp = st["temp"].double()[request][:, None]
    greedy = torch.zeros(st["logits"].shape, dtype=torch.float64, device=DEV)
    greedy.scatter_(1, st["logits"].argmax(1, keepdim=True), 1.0)
    p = torch.where(temp > 0, torch.softmax(st["logits"].double() / torch.where(temp > 0, temp, 1.0), 1), greedy)
    at = torch.arange(rows, device=DEV)[place < count]  # the row that verifies each draft
    p_x = p[at].gather(1, drafts[:, None]).squeeze(1)
    q_x = torch.ones_like(p_x) if st["q"] is None else st["q"].gather(1, drafts[:, None]).squeeze(1).double()
    refused = torch.zeros(rows, dtype=torch.int64, device=DEV)
    refused[at] = (st["u"].double() * q_x >= p_x).long()
    total = refused.cumsum(0)
    before = (total - refused)[off[:-1]][request]
    taken = (total - before == 0) & (place < count)  # every draft up to this one accepted
    accepted = torch.zeros(requests, dtype=torch.int64, device=DEV).index_add_(0, request, taken.long())
    last = off[:-1] + accepted  # the row that the final token comes from
    w = p[last]
    short = accepted < off[1:] - off[:-1] - 1  # a draft was refused there
    of = (last - torch.arange(requests, device=DEV)).clamp(max=max(0, len(drafts) - 1))
    if len(drafts):
        if st["q"] is None:
            q = torch.zeros_like(w).scatter_(1, drafts[of][:, None], 1.0)
        else:
            q = st["q"][of].double()
        rest = (w - q).clamp(min=0)
        w = torch.where(short[:, None] & (rest.sum(1, keepdim=True) > 0), rest, w)
    sums = w.cumsum(1)
    at_u = st["last"].double()[:, None] * sums[:, -1:]
    final = torch.minimum((sums <= at_u).sum(1), (sums < sums[:, -1:]).sum(1))
    tokens = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    mine = torch.zeros(rows, dtype=torch.int32, device=DEV)
    mine[at] = st["tokens"]
    tokens = torch.where(taken, mine, tokens)
    tokens[last] = final.to(torch.int32)
    return [accepted.to(torch.int32), tokens]


def work(case):
    if case["kind"] == "adapters":
        ns, k, rows, size = _ns(case), case["k"], case["rows"], DTYPE[case["dtype"]].itemsize
        used = min(case["slots"], case["requests"])
        rank = sum(_ranks(case)) / case["slots"]
        low = sum(rank * (k + n) for n in ns)
        return {"bytes": sum(ns) * k * ROW_BYTES[case["type"]] + used * low * size + 4 * rows * (k + sum(ns) + 1),
                "flops": 2.0 * rows * (sum(ns) * k + low)}
    if case["kind"] == "norm":
        planes = 1 + _has_sum(case) + case["residual"] + case["pre"] + (case["gate"] == "full")
        n = case["rows"] * case["k"]
        return {"bytes": 4 * (n * planes + case["k"] * (case["post"] + case["pre"] + (case["gate"] == "channel"))),
                "flops": n * (2 + 4 * case["post"] + 4 * case["pre"])}
    counts, vocab = _draft_counts(case), case["vocab"]
    rows = sum(counts) + case["requests"]
    return {"bytes": 4 * vocab * (rows + (case["requests"] if case["probs"] else 0)) + 16 * rows, "flops": 4.0 * rows * vocab}


# ------------------------------------------------------------------------------------------------- in 64 bits

def _exact_weight(type_, blocks, n, k):
    """[n][k] in 64 bits, one sub-block of every super-block after the other."""
    if type_ == Q8:
        return blocks[0].double().view(n, k) * blocks[1].double().repeat_interleave(32).view(n, k)
    b = blocks.view(n * k // 256, -1)
    f16 = lambda i: b[:, i:i + 2].contiguous().view(torch.float16).double()  # noqa: E731
    out = torch.empty(b.shape[0], 256, dtype=torch.float64, device=DEV)
    if type_ == Q4K:
        d, dmin = f16(0), f16(2)
        for j in range(8):
            if j < 4:
                sc, m = b[:, 4 + j] % 64, b[:, 8 + j] % 64
            else:
                sc = b[:, 8 + j] % 16 + b[:, j] // 64 * 16
                m = b[:, 8 + j] // 16 + b[:, 4 + j] // 64 * 16
            byte = b[:, 16 + 32 * (j // 2):48 + 32 * (j // 2)]
            quant = byte // 16 if j % 2 else byte % 16
            out[:, 32 * j:32 * j + 32] = d * sc.double()[:, None] * quant.double() - dmin * m.double()[:, None]
        return out.view(n, k)
    d, scales = f16(208), b[:, 192:208].contiguous().view(torch.int8).double()
    for j in range(8):  # 32 weights each: half j // 4, quarter j % 4
        half, quarter = j // 4, j % 4
        low = b[:, 64 * half + 32 * (quarter % 2):64 * half + 32 * (quarter % 2) + 32]
        low = low // 16 if quarter >= 2 else low % 16
        high = b[:, 128 + 32 * half:160 + 32 * half] // 4 ** quarter % 4
        quant = low.double() + 16 * high.double() - 32
        out[:, 32 * j:32 * j + 32] = quant * d * scales[:, 2 * j:2 * j + 2].repeat_interleave(16, 1)
    return out.view(n, k)


def _exact_q8(x, block):
    """The 8-bit activation is defined in 32-bit steps (scale, its reciprocal, the product); only its value is widened."""
    v = x.reshape(-1, block)
    top = v.abs().max(1).values
    scale = (top.double() / 127).float()
    inverse = torch.where(scale > 0, (1 / scale.double()).float(), torch.zeros_like(scale))
    quant = (v * inverse[:, None]).double().round().clamp(-127, 127)
    return (quant * scale.double()[:, None]).view(x.shape)


def _exact_adapters(case, seed):
    t = _adapter_inputs(case, seed)
    out = []
    for i, n in enumerate(_ns(case)):
        y = _exact_q8(t["x"], 32 if case["type"] == Q8 else 256) @ _exact_weight(case["type"], t["blocks"][i], n, case["k"]).t()
        for slot, rank in enumerate(_ranks(case)):
            rows = (t["slot"] == slot).nonzero().squeeze(1)
            if len(rows):
                low = t["x"][rows].double() @ t["a"][i][slot, :rank].double().t()
                y[rows] += float(t["scale"][slot]) * (low @ t["b"][i][slot, :, :rank].double().t())
        out.append(y if t["bias"] is None else y + t["bias"][i].double())
    return out


def _exact_norm(case, seed):
    t = _norm_inputs(case, seed)

    def normed(v, p):
        weight, bias = p
        if case["norm"] == "layer":
            var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
            return (v - mean) / (var + 1e-5).sqrt() * weight.double() + bias.double()
        return v / ((v * v).sum(1, keepdim=True) / case["k"] + 1e-5).sqrt() * weight.double()

    v = t["y"].double()
    if t["post"]:
        v = normed(v, t["post"])
    if t["gate"] is not None:
        v = v * (t["gate"].double().view(-1, 1) if case["gate"] == "row" else t["gate"].double())
    v = v * case["scale"]
    if t["h"] is not None:
        v = v + t["h"].double()
    return [v if _has_sum(case) else None, normed(v, t["pre"]) if t["pre"] else None]


def _exact_verify(case, seed):
    t = {k: None if v is None else v.cpu() for k, v in _verify_inputs(case, seed).items()}
    off, accepted, tokens = t["off"].tolist(), [], []
    for r in range(case["requests"]):
        n, out = off[r + 1] - off[r] - 1, []
        for i in range(n + 1):
            row = t["logits"][off[r] + i].double()
            if t["temp"][r] > 0:
                e = torch.exp((row - row.max()) / t["temp"][r].double())
                p = e / e.sum()
            else:
                p = torch.zeros_like(row)
                p[int(row.argmax())] = 1
            if i == n:
                w = p
                break
            d = off[r] - r + i
            x = int(t["tokens"][d])
            if t["q"] is None:
                q = torch.zeros_like(p)
                q[x] = 1
            else:
                q = t["q"][d].double()
            if t["u"][d].double() * q[x] < p[x]:
                out.append(x)
                continue
            w = torch.clamp(p - q, min=0)
            w = w if w.sum() > 0 else p
            break
        run_sum = w.cumsum(0)
        over = (run_sum > t["last"][r].double() * run_sum[-1]).nonzero()
        out.append(int(over[0]) if len(over) else int(w.nonzero()[-1]))
        accepted.append(len(out) - 1)
        tokens += out + [-1] * (n + 1 - len(out))
    return [torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)]


def exact(case, seed):
    return {"adapters": _exact_adapters, "norm": _exact_norm, "verify": _exact_verify}[case["kind"]](case, seed)
