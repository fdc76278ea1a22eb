"""The keys and values of a server's requests in a paged cache, measured: what lies between a block's q/k/v and output projections.

Kinds of case (the dict's "kind"):
  append    new tokens' keys into their requests' pages, turned by their positions (one axis, or time, height and width),
            rounded to the cache's type; values beside them; queries turned by the same angles
  attend    attention of each request's new tokens over its pages, causal among the new ones, optionally over a window
  selected  the same over a few pages a token and key head: its own, and those whose mean key fits its queries best

Sizes follow this repository's benchmark and tests (32 query and 8 key heads of 128); drawn cases spread them over heads of 64 to 256,
1 to 4100 new tokens, contexts from none to 131072, pages of 32 to 256 tokens, caches in fp16, bf16 and 8-bit integers (a scale for each
token and head, absmax / 127, ties to even). Queries, keys, values and outputs are fp32 in device memory.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}


# ---------------------------------------------------------------------------------------------------- the cases

def _case(name, kind, type_, requests, rows, context, heads=32, kv_heads=8, dim=128, page=64, ragged=False, window=0, top=0,
          style="pairs", axes=1, rotary=0):
    return {"name": name, "kind": kind, "type": type_, "requests": requests, "rows": rows, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged, "window": window, "top": top, "style": style,
            "axes": axes, "rotary": rotary or dim}


def listed():
    return [
        # One token of one request goes into the cache: the shortest call.
        _case("append_1row", "append", "f16", 1, 1, 4001),
        # Two images of 1297 patches in all behind their prompts: positions in time, height and width.
        _case("append_image_1297rows", "append", "bf16", 2, 1297, 300, style="halves", axes=3, ragged=True),
        # A prefill step of five prompts: the largest.
        _case("append_prefill_4096rows", "append", "f16", 5, 4096, 0, ragged=True),
        # One token of one request over a short conversation, where latency counts.
        _case("attend_1row", "attend", "f16", 1, 1, 1499),
        # A decode step of 64 requests of uneven lengths.
        _case("attend_decode_64rows", "attend", "f16", 64, 64, 8191, ragged=True),
        # Twelve requests' last tokens and four drafted ones each, over long documents in an 8-bit cache.
        _case("attend_drafts_60rows", "attend", "i8", 12, 60, 24000, ragged=True),
        # A chunk of a long prompt: 512 tokens over what came before.
        _case("attend_chunk_512rows", "attend", "bf16", 1, 512, 16000),
        # Three prompts of 4100 tokens in all, from their start: the largest.
        _case("attend_prefill_4100rows", "attend", "f16", 3, 4100, 0, ragged=True),
        # One token of one request over 131072, 32 pages of 64.
        _case("selected_1row", "selected", "f16", 1, 1, 131071, top=32),
        # A decode step of 24 requests over long documents in an 8-bit cache.
        _case("selected_decode_24rows", "selected", "i8", 24, 24, 32767, top=16, ragged=True),
        # A short chunk of one request over a long document, other pages for each token.
        _case("selected_chunk_130rows", "selected", "bf16", 1, 130, 20000, top=24),
    ]


def _logint(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "selected"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 128), (32, 32, 128), (16, 2, 64), (28, 4, 128), (8, 4, 256), (14, 2, 64), (40, 8, 128),
                                       (16, 16, 96)])
    page = rng.choice([32, 64, 64, 128, 256])
    style, ragged = rng.choice(["pairs", "halves"]), rng.random() < 0.6
    if kind == "append":
        rows = _logint(rng, 1, 4000)
        c = _case("", kind, rng.choice(["f16", "bf16"]), min(rows, _logint(rng, 1, 48)), rows, rng.choice([0, _logint(rng, 1, 8000)]), heads,
                  kv_heads, dim, page, ragged, style=style, axes=rng.choice([1, 1, 3]), rotary=rng.choice([dim, dim, dim // 2]))
    else:
        type_ = rng.choice(["f16", "bf16", "i8"])
        requests = _logint(rng, 1, 64)
        rows = requests * (1 if rng.random() < 0.4 else _logint(rng, 1, 1024 if kind == "attend" else 32))
        c = _case("", kind, type_, requests, rows, _logint(rng, 40, 131000), heads, kv_heads, dim, page, ragged,
                  window=rng.choice([0, 0, 0, 1024, 4000]) if kind == "attend" else 0,
                  top=_logint(rng, 2, 48) if kind == "selected" else 0)
        # no longer than the largest listed calls, and no more beside it in the plain form
        while work(c)["flops"] > 1.2e11 or _plain_scores(c) > 1.4e9 or work({**c, "kind": "attend"})["bytes"] > 1.2e9:
            if c["rows"] >= 2 * c["requests"]:
                c["rows"] //= 2
            elif c["requests"] > 1:
                c["requests"] //= 2
                c["rows"] = c["requests"]
            else:
                c["context"] //= 2
    del c["name"]
    return c


def _counts(c):
    """New tokens of each request."""
    r = c["requests"]
    weight = [1 + (3 * i) % 4 if c["ragged"] else 1 for i in range(r)]
    spare, done, out = c["rows"] - r, 0, []
    for i in range(r):
        upto = spare * sum(weight[:i + 1]) // sum(weight)
        out.append(1 + upto - done)
        done = upto
    return out


def _contexts(c):
    """Tokens that each request has in the cache before them."""
    return [c["context"] * (1 + (5 * i) % 8) // 8 if c["ragged"] and c["requests"] > 1 else c["context"] for i in range(c["requests"])]


def _plain_scores(c):
    """Scores that the plain form holds, requests padded to the longest."""
    return c["requests"] * c["heads"] * max(_counts(c)) * (max(_contexts(c)) + max(_counts(c)))


# ------------------------------------------------------------------------------------------------- what it holds

def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + part)


def _inputs(c, seed):
    gen = _gen(seed, 3)
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    order = torch.randperm(c["requests"], generator=gen, device=DEV).tolist()
    counts, contexts = [_counts(c)[i] for i in order], [_contexts(c)[i] for i in order]
    lengths = [n + m for n, m in zip(counts, contexts)]
    need = [-(-n // c["page"]) for n in lengths]
    t = {"rows": c["rows"], "width": max(need), "pool": sum(need) + 3, "counts": counts, "contexts": contexts}
    # each request's pages lie anywhere in the pool
    pages = torch.randperm(t["pool"], generator=gen, device=DEV).to(torch.int32)[:sum(need)]
    held = torch.arange(t["width"], device=DEV)[None] < torch.tensor(need, device=DEV)[:, None]
    t["tables"] = torch.full(held.shape, -1, dtype=torch.int32, device=DEV)
    t["tables"][held] = pages
    t["off"] = torch.tensor([0] + counts, device=DEV).cumsum(0).to(torch.int32)
    t["len"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    hk, d = c["kv_heads"], c["dim"]
    t["q"] = randn(c["rows"], c["heads"] * d) * 1.3
    if c["kind"] == "append":
        half = c["rotary"] // 2
        t["freq"] = (500000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)).float()
        t["k"], t["v"] = randn(c["rows"], hk * d), randn(c["rows"], hk * d)
        t["axis"] = t["pos"] = None
        if c["axes"] > 1:  # a quarter of the pairs for the time, the others for height and width; patches in rows of 31
            t["axis"] = (torch.arange(half, device=DEV) * 8 // (3 * half)).clamp(max=2).to(torch.int32)
            i = torch.cat([torch.arange(n, device=DEV) for n in counts])
            first = torch.cat([torch.full((n,), m, device=DEV) for n, m in zip(counts, contexts)])
            t["pos"] = torch.stack([first, first + i // 31, first + i % 31]).to(torch.int32)
        return t
    # stored keys: neighbours are alike, and some channels are far from zero
    total = sum(lengths)
    t["k"] = randn(total, hk, d) + 0.7 * randn(total // 64 + 1, hk, d).repeat_interleave(64, 0)[:total] + 0.5 * randn(hk, d)
    t["v"] = randn(total, hk, d) * 0.8 + 0.2
    t["at"] = torch.cat([torch.arange(n, device=DEV) for n in lengths])  # each stored token's place in its request
    t["of"] = torch.repeat_interleave(torch.arange(c["requests"], device=DEV), t["len"], output_size=total)
    return t


def _codes(x):
    """8-bit integers and their scale for each token and head, in 32-bit steps."""
    s = x.abs().amax(-1, keepdim=True)
    s = s / torch.full_like(s, 127.0)
    inv = torch.where(s > 0, torch.ones_like(s) / s, torch.zeros_like(s))
    return torch.round(x * inv).clamp(-127, 127).to(torch.int8), s


def _stored(c, t, x):
    """[pool][page][kv_heads][dim] of the stored tokens in the cache's type (8-bit: with the scales)."""
    slot = t["tables"].long()[t["of"], t["at"] // c["page"]] * c["page"] + t["at"] % c["page"]
    flat = lambda v, dt: torch.zeros(t["pool"] * c["page"], *v.shape[1:], dtype=dt, device=DEV).index_copy_(0, slot, v).view(  # noqa: E731
        t["pool"], c["page"], *v.shape[1:])
    if c["type"] == "i8":
        q, s = _codes(x)
        return flat(q, torch.int8), flat(s, torch.float32)
    return (flat(x.to(DTYPE[c["type"]]), DTYPE[c["type"]]),)


def _value(planes, at=None):
    """What stored planes stand for, in 32 bits; of the pages `at` only."""
    planes = [p if at is None else p[at] for p in planes]
    return planes[0].float() if len(planes) == 1 else planes[0].float() * planes[1]


def prepare(case, seed):
    st, t = dict(case), _inputs(case, seed)
    st.update({k: t[k] for k in ("tables", "off", "len", "q", "width", "pool")}, n=max(t["counts"]))
    if case["kind"] == "append":
        st.update({k: t[k] for k in ("k", "v", "freq", "axis", "pos")})
        if not own:
            st["cache"] = [torch.zeros(t["pool"], case["page"], case["kv_heads"], case["dim"], dtype=DTYPE[case["type"]], device=DEV)
                           for _ in "kv"]
    elif not own:
        st["kc"], st["vc"] = _stored(case, t, t["k"]), _stored(case, t, t["v"])
        if case["kind"] == "selected":  # kept with the cache: the sum of each page's keys
            st["sums"] = _value(st["kc"]).double().sum(1).float()
    if own:
        _prepare_own(st, case, t)
    return st


def _prepare_own(st, c, t):
    """What a server keeps: the cache with what was appended before, outputs and the prepared call."""
    import overfit_amd as ov

    ctx = ov.default_context()
    type_ = {"f16": ov.TYPE_F16, "bf16": ov.TYPE_BF16, "i8": ov.TYPE_I8}[c["type"]]
    cache = st["cache"] = ov.KvCache(c["kv_heads"], c["dim"], c["page"], t["pool"], type_, sums=c["kind"] == "selected")
    new = lambda *s, dt=torch.float32: torch.empty(s, dtype=dt, device=DEV)  # noqa: E731
    if c["kind"] == "append":
        rope = ov.Rope(st["freq"], st["style"], pair_axes=st["axis"])
        q_out = new(c["rows"], c["heads"] * c["dim"])
        st["out"] = [q_out, cache.key_view(), cache.value_view()]
        st["call"] = ctx.bind_kv_append_dev(cache, st["k"], st["v"], st["off"], st["len"], st["tables"], q=st["q"], q_out=q_out,
                                            rope=rope, positions=st["pos"])
        return
    first = 0
    for r, (n, m) in enumerate(zip(t["counts"], t["contexts"])):
        for at in range(0, n + m, 32768):
            upto = min(n + m, at + 32768)
            one = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
            ov.kv_append(cache, t["k"][first + at:first + upto], t["v"][first + at:first + upto], one([0, upto - at]), one([upto]),
                         t["tables"][r:r + 1])
        first += n + m
    out = new(c["rows"], c["heads"] * c["dim"])
    if c["kind"] == "attend":
        st["out"] = [out]
        st["call"] = ctx.bind_attend_dev(cache, st["q"], st["off"], st["len"], st["tables"], out, window=c["window"], max_rows=st["n"])
    else:
        st["out"] = [out, new(c["rows"], c["kv_heads"], c["top"], dt=torch.int32)]
        st["call"] = ctx.bind_attend_selected_dev(cache, st["q"], st["off"], st["len"], st["tables"], c["top"], out, pages=st["out"][1],
                                                  max_rows=st["n"])


def run(st):
    if own:
        st["call"]()
        return st["out"]
    return _plain_append(st) if st["kind"] == "append" else _plain_attend(st)


# --------------------------------------------------------------------------------------------------- plain forms

def _requests(st):
    """(request, place among its new tokens) of every row."""
    off = st["off"].long()
    of = torch.repeat_interleave(torch.arange(st["requests"], device=DEV), off[1:] - off[:-1], output_size=st["rows"])
    return of, torch.arange(st["rows"], device=DEV) - off[of]


def _plain_append(st):
    of, i = _requests(st)
    off, page, rot, half = st["off"].long(), st["page"], st["rotary"], st["rotary"] // 2
    at = st["len"].long()[of] - (off[1:] - off[:-1])[of] + i
    # angles in 64 bits
    pos = at[:, None].expand(-1, half) if st["pos"] is None else st["pos"].long()[st["axis"].long()].t()
    angle = pos.double() * st["freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, heads):
        x = x.view(st["rows"], heads, st["dim"])
        a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if st["style"] == "pairs" else (x[..., :half], x[..., half:rot])
        a, b = a * cos - b * sin, b * cos + a * sin
        return torch.cat([torch.stack([a, b], -1).flatten(-2) if st["style"] == "pairs" else torch.cat([a, b], -1), x[..., rot:]], -1)

    slot = (st["tables"].long()[of, at // page], at % page)
    k, v = st["cache"]
    k[slot] = turned(st["k"], st["kv_heads"]).to(k.dtype)
    v[slot] = st["v"].view(st["rows"], st["kv_heads"], st["dim"]).to(v.dtype)
    q = turned(st["q"], st["heads"]).view(st["rows"], -1)
    pool, d = st["pool"], st["dim"]
    # a page's tokens and a head's channels in the groups that the kernels hold together
    return [q, k.view(pool, page // 32, 2, 16, -1, d // 32, 4, 8), v.view(pool, page // 32, 2, 4, 4, st["kv_heads"], d // 16, 16)]


def _plain_attend(st):
    of, i = _requests(st)
    off, n, d, hk = st["off"].long(), st["n"], st["dim"], st["kv_heads"]
    r, g, width, page = st["requests"], st["heads"] // hk, st["width"], st["page"]
    q = torch.zeros(r, n, hk, g, d, device=DEV)
    q[of, i] = st["q"].view(-1, hk, g, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(r, hk, n * g, d)
    at = st["tables"].long().clamp(min=0)
    gathered = lambda c: _value(c, at).view(r, width * page, hk, d).permute(0, 2, 1, 3).contiguous()  # noqa: E731
    scores = (q @ gathered(st["kc"]).transpose(2, 3) / math.sqrt(d)).view(r, hk, n, g, width * page)
    place = (st["len"].long() - (off[1:] - off[:-1]))[:, None] + torch.arange(n, device=DEV)  # [r][n]
    key = torch.arange(width * page, device=DEV)
    seen = (key <= place[..., None]) & (key < st["len"].long()[:, None, None])
    if st["window"]:
        seen &= key > place[..., None] - st["window"]
    seen = seen[:, None]
    if st["kind"] == "selected":
        # each page's fit in 64 bits: one fit falls between two others
        sums = st["sums"][at].double().permute(0, 2, 3, 1).contiguous()  # [r][hk][d][width]
        fit = (q.double() @ sums).view(r, hk, n, g, width).amax(3)
        whole = torch.arange(width, device=DEV)
        mine = (place // page)[:, None, :, None]
        order = torch.where(whole < mine, fit, -math.inf).sort(dim=-1, descending=True, stable=True)[1][..., :st["top"] - 1]
        keep = torch.zeros(fit.shape, dtype=torch.bool, device=DEV).scatter_(-1, order, order < mine) | (whole == mine)
        seen = seen & keep.repeat_interleave(page, -1)
    scores = scores.masked_fill(~seen[:, :, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = (p.view(r, hk, n * g, -1) @ gathered(st["vc"])).view(r, hk, n, g, d).permute(0, 2, 1, 3, 4)
    out = out[of, i].reshape(st["rows"], -1)
    if st["kind"] == "attend":
        return [out]
    pages = torch.where(keep, whole, width).sort(-1)[0][..., :st["top"]]
    pages = torch.nn.functional.pad(pages, (0, st["top"] - pages.shape[-1]), value=width)
    return [out, torch.where(pages < width, pages, -1).permute(0, 2, 1, 3)[of, i].to(torch.int32)]


def work(case):
    c, counts, contexts = case, _counts(case), _contexts(case)
    hk, d, heads, rows = c["kv_heads"], c["dim"], c["heads"], c["rows"]
    token = 2 * hk * (d * DTYPE[c["type"]].itemsize + (4 if c["type"] == "i8" else 0))
    if c["kind"] == "append":
        return {"bytes": rows * (8 * heads * d + 8 * hk * d + token), "flops": 3.0 * rows * (heads + hk) * c["rotary"]}
    flops, read = 0.0, 0
    for n, m in zip(counts, contexts):
        if c["kind"] == "attend":
            most = c["window"] or m + n
            short = max(0, min(n, most - m))  # rows that see all before them
            flops += 4.0 * heads * d * (short * m + short * (short + 1) / 2 + (n - short) * min(most, m + n))
            read += token * min(m + n, most + n)
        else:
            keys = min(m + n, c["top"] * c["page"])
            flops += n * heads * d * (4.0 * keys + 2.0 * (m // c["page"]))
            read += token * min(m + n, n * keys) + 4 * hk * d * ((m + n) // c["page"])
    return {"bytes": read + 8 * rows * heads * d, "flops": flops}


# ------------------------------------------------------------------------------------------------- in 64 bits

def _exact_append(c, t):
    hk, h, d, rot, page = c["kv_heads"], c["heads"], c["dim"], c["rotary"], c["page"]
    q, k = t["q"].double().view(-1, h, d).clone(), t["k"].double().view(-1, hk, d).clone()
    cache = torch.zeros(2, t["pool"], page, hk, d, dtype=torch.float64, device=DEV)
    i0 = 0
    for r, (n, m) in enumerate(zip(t["counts"], t["contexts"])):
        rows = slice(i0, i0 + n)
        for pair in range(rot // 2):
            place = torch.arange(m, m + n, device=DEV) if t["pos"] is None else t["pos"][int(t["axis"][pair]), rows]
            turn = torch.polar(torch.ones(n, dtype=torch.float64, device=DEV), place.double() * float(t["freq"][pair]))[:, None]
            x, y = (2 * pair, 2 * pair + 1) if c["style"] == "pairs" else (pair, pair + rot // 2)
            for z in (q, k):
                w = torch.complex(z[rows, :, x], z[rows, :, y]) * turn
                z[rows, :, x], z[rows, :, y] = w.real, w.imag
        at = torch.arange(m, m + n, device=DEV)
        where = t["tables"][r].long()[at // page], at % page
        cache[0][where], cache[1][where] = k[rows], t["v"].double().view(-1, hk, d)[rows]
        i0 += n
    return [q.view(c["rows"], -1), cache[0].view(t["pool"], page // 32, 2, 16, hk, d // 32, 4, 8),
            cache[1].view(t["pool"], page // 32, 2, 4, 4, hk, d // 16, 16)]


def _exact_stored(c, x):
    """One request's keys or values as the cache holds them; what 8 bits hold is defined in 32-bit steps."""
    if c["type"] != "i8":
        return x.to(DTYPE[c["type"]]).double()
    top = x.abs().max(-1, keepdim=True).values
    scale = (top.double() / 127).float()
    inverse = torch.where(scale > 0, (1 / scale.double()).float(), torch.zeros_like(scale))
    return (x * inverse).double().round().clamp(-127, 127) * scale.double()


def _exact_attend(c, t):
    hk, h, d, page, top = c["kv_heads"], c["heads"], c["dim"], c["page"], c["top"]
    g = h // hk
    out = torch.empty(c["rows"], hk, g, d, dtype=torch.float64, device=DEV)
    chosen = torch.full((c["rows"], hk, top), -1, dtype=torch.int32, device=DEV)
    i0 = j0 = 0
    for n, m in zip(t["counts"], t["contexts"]):
        rows, keys = slice(i0, i0 + n), slice(j0, j0 + n + m)
        i0, j0 = i0 + n, j0 + n + m
        place, key = torch.arange(m, m + n, device=DEV)[:, None], torch.arange(m + n, device=DEV)[None]
        for a in range(hk):
            k, v = _exact_stored(c, t["k"][keys, a]), _exact_stored(c, t["v"][keys, a])
            hidden = key > place
            if c["window"]:
                hidden = hidden | (place - key >= c["window"])
            q = [t["q"][rows, (a * g + b) * d:(a * g + b + 1) * d].double() for b in range(g)]
            if top:
                full = (n + m) // page
                means = k[:full * page].view(full, page, d).sum(1).float().double()
                fit = torch.stack([x @ means.t() for x in q]).max(0).values
                before = torch.arange(full, device=DEV)[None] < place // page
                fit = fit.masked_fill(~before, -math.inf)
                best = torch.argsort(-fit, dim=1, stable=True)[:, :top - 1]
                lists = torch.cat([torch.where(before.gather(1, best), best, 1 << 30), place // page], 1).sort(1).values
                chosen[rows, a, :lists.shape[1]] = torch.where(lists < 1 << 30, lists, -1).to(torch.int32)
                taken = torch.zeros(n, -(-(n + m) // page) + 1, dtype=torch.bool, device=DEV)
                taken.scatter_(1, lists.clamp(max=taken.shape[1] - 1), True)
                hidden = hidden | ~taken.gather(1, (key // page).expand(n, -1))
            for b in range(g):
                s = (q[b] @ k.t() / math.sqrt(d)).masked_fill(hidden, -math.inf)
                out[rows, a, b] = torch.softmax(s, 1) @ v
    return [out.view(c["rows"], -1)] + ([chosen] if top else [])


def exact(case, seed):
    t = _inputs(case, seed)
    return _exact_append(case, t) if case["kind"] == "append" else _exact_attend(case, t)
