"""The measured work of a packed step's attention layers and of its end: the operators between the
q/k/v projections and the out projection, and the verification of drafted tokens after the lm_head.

Kinds of case, each one pass through one operator:

* ``heads`` -- queries and keys normed over each head and rotated by their rows' positions.
* ``cache`` -- the step's keys (normed and rotated) and values kept in 8 bits in a paged cache, its
  queries normed and rotated beside them, and the last tokens of each request read back.
* ``attend`` -- causal attention of the step's rows over that cache: query heads in groups on one
  key/value head, uneven requests, and a prefix that all requests may share.
* ``verify`` -- drafted tokens against the target's probabilities: how many of each request's are
  accepted, and the token that follows them, from given uniform random numbers.

Sizes are those of the library's workloads (q 24 heads and k, v 4 heads of 256: projections of 6144
and 1024 outputs; vocabulary 248320; verify steps of 8 x 8 rows, prompts of 2048) and odd ones of the
same form. With ``own`` false the operators are computed with elementary torch operations, with
``own`` true by the library's entry points.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
LEAST_SCALE = 2.0 ** -100


def listed():
    def heads(name, rows, q_heads, kv_heads, dim, rotary, dtype, padded=False):
        return {"name": name, "kind": "heads", "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rotary, "dtype": dtype, "padded": padded}

    def cache(name, requests, rows, longest, read, q_heads, kv_heads, dim, rotary, page, dtype, padded=False):
        return {"name": name, "kind": "cache", "requests": requests, "rows": rows, "longest": longest, "read": read,
                "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "page": page, "dtype": dtype,
                "padded": padded, "shared": 0, "uneven": False}

    def attend(name, requests, rows, longest, q_heads, kv_heads, dim, page, shared=0, uneven=False, padded=False):
        return {"name": name, "kind": "attend", "requests": requests, "rows": rows, "longest": longest, "q_heads": q_heads,
                "kv_heads": kv_heads, "dim": dim, "page": page, "shared": shared, "uneven": uneven, "padded": padded}

    def verify(name, requests, rows, vocab, dtype, draft, flat=False, padded=False):
        return {"name": name, "kind": "verify", "requests": requests, "rows": rows, "vocab": vocab, "dtype": dtype,
                "draft": draft, "flat": flat, "padded": padded}

    return [
        # One token of one request: all latency. Queries lie beside their gates in a wider projection.
        heads("heads_decode_1", 1, 24, 4, 256, 64, "bf16", padded=True),
        # A prompt, from fp32 projections.
        heads("heads_prompt_2048", 2048, 24, 4, 256, 64, "f32"),
        # A verify step: eight rows of eight requests each written, and 512 tokens a request read back.
        cache("cache_verify_64", 8, 64, 4096, 512, 24, 4, 256, 64, 256, "bf16", padded=True),
        # A prompt written and read back whole, odd pages, all of a head rotated.
        cache("cache_prompt_2000", 1, 2000, 2000, 2000, 16, 8, 128, 128, 96, "f32"),
        # One token of one request on a context of 4111: latency, few keys to share among the CUs.
        attend("attend_decode_1", 1, 1, 4111, 24, 4, 256, 256),
        # Sixty-four requests of one token, contexts from 800 to 8192.
        attend("attend_decode_64", 64, 64, 8192, 24, 4, 256, 256, uneven=True),
        # A verify step of 8 x 8 rows on long contexts.
        attend("attend_verify_64", 8, 64, 32768, 24, 4, 256, 256, uneven=True),
        # Sixteen requests of four drafted tokens on one prefix of 16384, up to 1024 tokens of their own.
        attend("attend_shared_64", 16, 64, 17408, 24, 4, 256, 256, shared=16384, uneven=True),
        # An odd batch: seven requests, uneven runs of rows, heads of 128 in groups of five, odd pages.
        attend("attend_odd_333", 7, 333, 2777, 10, 2, 128, 96, uneven=True, padded=True),
        # A chunk of a prompt: 2048 rows on 6144 tokens before them.
        attend("attend_prefill_2048", 1, 2048, 8192, 24, 4, 256, 256),
        # Seven drafted tokens of eight requests each against the draft's probabilities.
        verify("verify_64", 8, 64, 248320, "f32", "probabilities"),
        # A wide batch of tokens that a lookup drafted (no probabilities of theirs), on an odd vocabulary in bf16.
        verify("verify_lookup_256", 40, 256, 32003, "bf16", "lookup", padded=True),
    ]


def _between(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["heads", "cache", "attend", "attend", "attend", "verify"])
    if kind == "verify":
        vocab = _between(rng, 1000, 248320)
        rows = min(_between(rng, 2, 256), 64 * 248320 // vocab)
        return {"kind": kind, "requests": max(1, rows // rng.randint(1, 9)), "rows": rows, "vocab": vocab,
                "dtype": rng.choice(["f32", "bf16"]), "draft": rng.choice(["probabilities", "probabilities", "lookup"]),
                "flat": rng.random() < 0.3, "padded": rng.random() < 0.3}
    dim = rng.choice([64, 128, 256, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 7, 8])
    rotary = rng.choice([dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
    if kind == "heads":
        return {"kind": kind, "rows": _between(rng, 1, 2048), "q_heads": min(24, q_heads), "kv_heads": min(4, kv_heads),
                "dim": dim, "rotary": rotary, "dtype": rng.choice(["f32", "bf16"]), "padded": rng.random() < 0.3}
    page = rng.choice([32, 64, 96, 256, 32 * rng.randint(1, 16)])
    if kind == "cache":
        requests = _between(rng, 1, 64)
        rows = max(requests, _between(rng, 1, 2000))
        longest = -(-rows // requests) + _between(rng, 1, 4096)
        return {"kind": kind, "requests": requests, "rows": rows, "longest": longest,
                "read": min(longest, _between(rng, 1, max(1, 4096 // requests))), "q_heads": min(24, q_heads),
                "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "page": page, "dtype": rng.choice(["f32", "bf16"]),
                "padded": rng.random() < 0.3, "shared": 0, "uneven": rng.random() < 0.5}
    requests = _between(rng, 1, 64)
    rows = requests * rng.randint(1, 8) if rng.random() < 0.6 else max(requests, _between(rng, 1, 1024))
    mean = -(-rows // requests)
    longest = 2 * mean + _between(rng, 1, max(64, min(32768, 8 * 32768 // requests)))
    # (Rows times keys as the prompt's chunk has, and no more.)
    while longest > 2 * mean + 64 and longest * rows * q_heads * dim > 2048 * 7168 * 24 * 256:
        longest = 2 * mean + (longest - 2 * mean) // 2
    shared = 0
    if requests > 1 and rng.random() < 0.3:
        shared = longest // page * page
        longest += 2 * mean + _between(rng, 1, 1024)
    return {"kind": kind, "requests": requests, "rows": rows, "longest": longest, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "shared": shared, "uneven": rng.random() < 0.6, "padded": rng.random() < 0.3}


# ---- the step's shape, from the case alone -------------------------------------------------------


def _spread(count, salt):
    """`count` numbers in [0, 1) that lie apart from each other."""
    return [(0.5 + (i + salt) * 0.6180339887498949) % 1.0 for i in range(count)]


def _runs(case):
    """How many rows each request has: the same, or uneven runs of one at least."""
    rows, requests = case["rows"], case["requests"]
    if not case.get("uneven", True) or rows % requests == 0:
        return [rows // requests + (r < rows % requests) for r in range(requests)]
    cuts = sorted(1 + int(x * (rows - requests)) for x in _spread(requests - 1, 3))
    cuts = [c + i for i, c in enumerate(cuts)]  # (apart from each other)
    return [b - a for a, b in zip([0] + cuts, cuts + [rows])]


def _lengths(case):
    """How many tokens each request has in the cache after the step, its own rows among them."""
    runs, shared = _runs(case), case["shared"]
    if not case["uneven"]:
        return [max(case["longest"], shared + n) for n in runs]
    return [max(shared + n, shared + int((case["longest"] - shared) * (0.1 + 0.9 * x))) for n, x in zip(runs, _spread(len(runs), 0))]


# ---- inputs, from the seed alone ----------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000 + salt)


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _rows_of(t, padded):
    """`t` as rows of a wider buffer, where the case asks for that."""
    if not padded:
        return t
    wide = torch.zeros(t.shape[0], t.shape[1] + 24, dtype=t.dtype, device=t.device)
    wide[:, : t.shape[1]] = t
    return wide[:, : t.shape[1]]


def _heads_of(gen, rows, heads, dim, dtype, padded):
    """[rows, heads, dim] as a projection gives it; `padded`: each head beside a gate of its size."""
    x = (_normal(gen, rows, heads, dim) * 1.5).to(DTYPES[dtype])
    if not padded:
        return x
    wide = torch.zeros(rows, heads, 2 * dim, dtype=x.dtype, device=x.device)
    wide[..., :dim] = x
    return wide[..., :dim]


def _rotation(case, seed):
    """Norm weights of q and k in bf16, and the rotation's frequencies."""
    gen, half = _gen(seed, 1), case["rotary"] // 2
    weights = [(1.0 + 0.3 * _normal(gen, case["dim"])).to(torch.bfloat16) for _ in range(2)]
    steps = torch.arange(half, dtype=torch.float64, device="cuda") / half
    return weights[0], weights[1], (1.0e7 ** -steps).float()


def _head_inputs(case, seed):
    gen = _gen(seed, 2)
    q, k = (_heads_of(gen, case["rows"], n, case["dim"], case["dtype"], case["padded"]) for n in (case["q_heads"], case["kv_heads"]))
    q_weight, k_weight, frequencies = _rotation(case, seed)
    positions = torch.randint(0, 262144, (case["rows"],), dtype=torch.int32, device="cuda", generator=gen)
    return {"q": q, "k": k, "q_weight": q_weight, "k_weight": k_weight, "frequencies": frequencies, "positions": positions}


def _packed_inputs(case, seed):
    """Where the rows lie: starts of the requests' runs, lengths, and a table of pages in no order. Requests share
    the pages of the shared prefix, and leave a page or two of the cache free."""
    runs, lengths, page = _runs(case), _lengths(case), case["page"]
    requests, common = len(runs), case["shared"] // page
    wide = max(-(-n // page) for n in lengths)
    own_pages = [-(-n // page) - common for n in lengths]
    pages = common + sum(own_pages) + 2
    order = torch.randperm(pages, device="cuda", generator=_gen(seed, 3)).to(torch.int32)
    first = torch.tensor([common + sum(own_pages[:r]) for r in range(requests)], device="cuda")
    column = torch.arange(wide, device="cuda")
    index = torch.where(column < common, column, first[:, None] + column - common)
    last = torch.tensor([common + n for n in own_pages], device="cuda")
    table = torch.where(column < last[:, None], order[index.clamp(max=pages - 1)], -1)
    starts = torch.tensor([sum(runs[:r]) for r in range(requests + 1)], dtype=torch.int32, device="cuda")
    return {"starts": starts, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            "table": table.to(torch.int32), "pages": pages}


def _history(case, seed):
    """What the cache holds before the measured pass, by page: keys and values in bf16, some tokens much smaller."""
    gen, pages = _gen(seed, 4), case["pages"]
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    size = torch.exp(0.5 * _normal(gen, pages, case["page"], case["kv_heads"], 1))
    return (_normal(gen, *shape) * size).to(torch.bfloat16), (_normal(gen, *shape) * size.flip(0)).to(torch.bfloat16)


def _logits(case, seed):
    """A bulk of unlikely tokens and, unless `flat`, a head of a few dozen likely ones that decays."""
    rows, vocab = case["rows"], case["vocab"]
    gen = _gen(seed, 5)
    logits = 2.0 * _normal(gen, rows, vocab)
    if not case["flat"]:
        head = min(vocab, 48)
        at = torch.randint(0, vocab, (rows, head), device="cuda", generator=gen)
        bonus = 15.0 - 9.0 * torch.rand(rows, head, device="cuda", generator=gen).sqrt()
        logits.scatter_reduce_(1, at, bonus, "amax")  # (a place drawn twice: the larger, whatever the order)
    return logits


def _verify_inputs(case, seed):
    """The step's tokens: of each request the last one it was given, then the drafted ones, each drawn by a draft whose
    logits are near the target's. Some requests are greedy."""
    rows, vocab, gen = case["rows"], case["vocab"], _gen(seed, 6)
    logits = _logits(case, seed)
    draft = torch.softmax(logits + 0.7 * _normal(gen, rows, vocab), 1)
    if case["draft"] == "lookup":
        drafted = (logits + 2.0 * _normal(gen, rows, vocab)).argmax(1)
    else:
        drafted = (draft / torch.empty_like(draft).exponential_(generator=gen)).argmax(1)
    tokens = torch.cat([drafted.new_zeros(1), drafted[:-1]]).to(torch.int32)  # (row m is judged at row m - 1)
    runs = _runs(case)
    starts = torch.tensor([sum(runs[:r]) for r in range(len(runs) + 1)], dtype=torch.int32, device="cuda")
    temperature = 0.6 + 0.6 * torch.rand(len(runs), device="cuda", generator=gen)
    greedy = torch.rand(len(runs), device="cuda", generator=gen) < 0.2
    return {"logits": _rows_of(logits.to(DTYPES[case["dtype"]]), case["padded"]), "tokens": tokens, "starts": starts,
            "uniforms": torch.rand(rows, device="cuda", generator=gen),
            "temperature": torch.where(greedy, torch.zeros_like(temperature), temperature),
            "draft": _rows_of(draft, case["padded"]) if case["draft"] == "probabilities" else None}


def _inputs(case, seed):
    if case["kind"] == "heads":
        return _head_inputs(case, seed)
    if case["kind"] == "verify":
        return _verify_inputs(case, seed)
    st = _packed_inputs(case, seed)
    st["history"] = _history(case | {"pages": st["pages"]}, seed)
    gen = _gen(seed, 7)
    if case["kind"] == "cache":
        for name, heads in (("q", case["q_heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"])):
            st[name] = _heads_of(gen, case["rows"], heads, case["dim"], case["dtype"], case["padded"])
        st["q_weight"], st["k_weight"], st["frequencies"] = _rotation(case, seed)
        reads = [min(case["read"], n) for n in _lengths(case)]
        st["read_starts"] = torch.tensor([sum(reads[:r]) for r in range(len(reads) + 1)], dtype=torch.int32, device="cuda")
        st["read_rows"] = sum(reads)
    else:
        st["q"] = _heads_of(gen, case["rows"], case["q_heads"], case["dim"], "bf16", case["padded"])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    rows = case["rows"]
    if case["kind"] == "verify":
        if own:  # the outputs and scratch that a serving program keeps between steps
            from splosh_amd import runtime as rt
            st["out"] = torch.empty(rows, dtype=torch.int32, device="cuda")
            st["accepted"] = torch.empty(case["requests"], dtype=torch.int32, device="cuda")
            st["workspace"] = torch.zeros(rt.verify_workspace_bytes(rows, case["vocab"], case["requests"]), dtype=torch.uint8,
                                          device="cuda")
        return st
    outputs = {"heads": ("q", "k"), "cache": ("q",), "attend": ("q",)}[case["kind"]]
    if own:
        for name in outputs:
            st[name + "_out"] = torch.empty(st[name].shape, dtype=torch.bfloat16, device="cuda")
    if case["kind"] == "heads":
        return st
    keys, values = st.pop("history")
    if own:
        from splosh_amd import runtime as rt
        st["cache"] = rt.Cache.empty(st["pages"], case["page"], case["kv_heads"], case["dim"], "cuda")
        st["packed"] = rt.Packed(st["starts"], st["lengths"], st["table"])
        # The history is written as one request of all the pages.
        whole = torch.arange(st["pages"], dtype=torch.int32, device="cuda")[None]
        count = st["pages"] * case["page"]
        ends = torch.tensor([0, count], dtype=torch.int32, device="cuda")
        rt.cache_write(st["cache"], rt.Packed(ends, ends[1:].clone(), whole), keys.flatten(0, 1), values.flatten(0, 1))
        if case["kind"] == "cache":
            st["read"] = rt.Packed(st["read_starts"], st["lengths"], st["table"])
            st["k_read"], st["v_read"] = (torch.empty(st["read_rows"], case["kv_heads"], case["dim"], dtype=torch.bfloat16,
                                                      device="cuda") for _ in range(2))
        else:
            need = rt.attend_workspace_bytes(st["cache"], st["packed"], rows, case["q_heads"], case["shared"])
            st["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    else:
        st["keys"], st["values"] = _plain_quantised(keys.float()), _plain_quantised(values.float())
    return st


# ---- the operators ------------------------------------------------------------------------------


def _plain_rotated(x, weight, frequencies, positions):
    """Norm over the head, then pairs (i, i + half) turned by position times frequency, angles in 64 bits."""
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    angle = positions.double()[:, None] * frequencies.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = frequencies.numel()
    a, b = y[..., :half], y[..., half : 2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half :]], -1)


def _plain_quantised(x):
    """(codes, scales) of vectors along the last dimension."""
    most = x.abs().amax(-1, keepdim=True)
    small = most / 127.0 < LEAST_SCALE
    codes = torch.where(small, x / LEAST_SCALE, x * 127.0 / torch.where(small, torch.ones_like(most), most))
    return codes.round().to(torch.int8), torch.where(small, torch.full_like(most, LEAST_SCALE), most / 127.0)


def _plain_places(starts, lengths, rows):
    """Each row's request and its position there."""
    row = torch.arange(rows, device=starts.device)
    request = torch.searchsorted(starts.long(), row, right=True) - 1
    return request, lengths[request] - starts[request + 1] + row


def _plain_slots(st, starts, rows):
    """(page, place in it, position) of each row's token."""
    request, position = _plain_places(starts, st["lengths"], rows)
    page = st["case"]["page"]
    return st["table"][request, position // page].long(), position % page, position


def _plain_cache(st):
    pages, place, position = _plain_slots(st, st["starts"], st["case"]["rows"])
    q = _plain_rotated(st["q"], st["q_weight"], st["frequencies"], position).to(torch.bfloat16)
    k = _plain_rotated(st["k"], st["k_weight"], st["frequencies"], position)
    for (codes, scales), x in ((st["keys"], k), (st["values"], st["v"].float())):
        codes[pages, place], scales[pages, place] = _plain_quantised(x)
    pages, place, _ = _plain_slots(st, st["read_starts"], st["read_rows"])
    return (q, *((codes[pages, place].float() * scales[pages, place]).to(torch.bfloat16) for codes, scales in (st["keys"], st["values"])))


def _plain_attend(st):
    """Every request's pages gathered, and its rows side by side: a product, a masked softmax, a product."""
    case, table = st["case"], st["table"].clamp(min=0).long()
    rows, heads, dim, group = case["rows"], case["kv_heads"], case["dim"], case["q_heads"] // case["kv_heads"]
    request, position = _plain_places(st["starts"], st["lengths"], rows)
    most = max(_runs(case))
    at = torch.arange(rows, device=table.device) - st["starts"][request]
    q = torch.zeros(len(table), most, heads, group, dim, device=table.device)
    q[request, at] = st["q"].float().reshape(rows, heads, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(len(table) * heads, most * group, dim)

    def gathered(codes, scales):
        x = codes[table].float().mul_(scales[table])  # [requests, pages, page, heads, dim]
        return x.flatten(1, 2).transpose(1, 2).reshape(len(table) * heads, -1, dim)

    score = torch.bmm(q, gathered(*st["keys"]).transpose(1, 2).contiguous()).mul_(dim ** -0.5)
    last = torch.full((len(table), most), -1, device=table.device)
    last[request, at] = position
    masked = torch.arange(score.shape[-1], device=table.device) > last[:, None, :, None, None]
    score = score.view(len(table), heads, most, group, -1).masked_fill_(masked, -math.inf).view_as(score)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    out = torch.bmm(weight, gathered(*st["values"])) / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = out.view(len(table), heads, most, group, dim).permute(0, 2, 1, 3, 4)[request, at]
    return out.reshape(rows, heads * group, dim).to(torch.bfloat16)


def _plain_verify(st):
    """In 64 bits: the sums decide between neighbouring tokens."""
    starts, tokens, u = st["starts"].long(), st["tokens"].long(), st["uniforms"].double()
    rows, vocab = st["logits"].shape
    row = torch.arange(rows, device=tokens.device)
    request = torch.searchsorted(starts, row, right=True) - 1
    temperature = st["temperature"].double()[request][:, None]
    logits = st["logits"].double()
    first = logits.argmax(1, keepdim=True)
    p = torch.softmax(logits / torch.where(temperature > 0, temperature, 1.0), 1)
    p = torch.where(temperature > 0, p, torch.zeros_like(p).scatter_(1, first, 1.0))
    last = row == starts[request + 1] - 1
    token = tokens[(row + 1).clamp(max=rows - 1)]
    q_token = st["draft"].double().gather(1, token[:, None])[:, 0] if st["draft"] is not None else 1.0
    accepted = (u * q_token < p.gather(1, token[:, None])[:, 0]) & ~last
    # How many rows from each start on are accepted: up to the first that is not.
    stop = torch.where(accepted, rows, row)
    stop = torch.full_like(starts[:-1], rows).scatter_reduce_(0, request, stop, "amin")
    count = stop - starts[:-1]
    p, drawn = p[stop], u[starts[1:] - 1]
    if st["draft"] is not None:
        q = st["draft"].double()[stop]
    else:
        q = torch.zeros_like(p).scatter_(1, token[stop][:, None], 1.0)
    rest = torch.where(last[stop][:, None], p, (p - q).clamp(min=0.0))
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    running = rest.cumsum(1)
    new = (running > drawn[:, None] * running[:, -1:]).to(torch.uint8).argmax(1)
    out = torch.where(row < stop[request], token, torch.where(row == stop[request], new[request], -1))
    return out.int(), count.int()


def _plain(st):
    kind = st["case"]["kind"]
    if kind == "heads":
        return [_plain_rotated(st[n], st[n + "_weight"], st["frequencies"], st["positions"]).to(torch.bfloat16) for n in ("q", "k")]
    return {"cache": _plain_cache, "attend": _plain_attend, "verify": _plain_verify}[kind](st)


def run(st):
    if not own:
        return _plain(st)
    from splosh_amd import runtime as rt
    kind = st["case"]["kind"]
    if kind == "heads":
        return rt.rotate_heads([st["q"], st["k"]], st["positions"], st["frequencies"], [st["q_weight"], st["k_weight"]], EPS,
                               outs=[st["q_out"], st["k_out"]])
    if kind == "cache":
        q = rt.cache_write(st["cache"], st["packed"], st["k"], st["v"], st["q"], st["frequencies"], st["k_weight"],
                           st["q_weight"], EPS, out=st["q_out"])
        return (q, *rt.cache_read(st["cache"], st["read"], k=st["k_read"], v=st["v_read"]))
    if kind == "attend":
        return rt.attend(st["q"], st["cache"], st["packed"], shared=st["case"]["shared"], out=st["q_out"], workspace=st["workspace"])
    return rt.verify(st["logits"], st["tokens"], st["starts"], st["uniforms"], st["temperature"], st["draft"], out=st["out"],
                     accepted=st["accepted"], workspace=st["workspace"])


# ---- what a pass cannot do without, and what it has to give ---------------------------------------


def work(case):
    rows = case["rows"]
    if case["kind"] == "verify":
        size, values = (4 if case["dtype"] == "f32" else 2), rows * case["vocab"]
        draft = case["requests"] * case["vocab"] * 4 if case["draft"] == "probabilities" else 0
        return {"bytes": values * size + draft + rows * 12 + case["requests"] * 12, "flops": 3 * values}
    q_heads, kv_heads, dim = case["q_heads"], case["kv_heads"], case["dim"]
    size = 2 if case.get("dtype", "bf16") == "bf16" else 4
    q, kv, token = rows * q_heads * dim, rows * kv_heads * dim, kv_heads * (dim + 4)
    if case["kind"] == "heads":
        return {"bytes": (q + kv) * (size + 2) + rows * 4, "flops": 8 * (q + kv)}
    if case["kind"] == "cache":
        read = sum(min(case["read"], n) for n in _lengths(case))
        return {"bytes": q * (size + 2) + 2 * kv * size + 2 * rows * token + 2 * read * (token + 2 * kv_heads * dim),
                "flops": 8 * q + 16 * kv + 2 * read * kv_heads * dim}
    runs, lengths = _runs(case), _lengths(case)
    tokens = case["shared"] + sum(n - case["shared"] for n in lengths)
    keys = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(runs, lengths))  # over all rows
    return {"bytes": 2 * q * 2 + 2 * tokens * token + sum(-(-n // case["page"]) for n in lengths) * 4,
            "flops": 4 * keys * q_heads * dim}


def _exact_rotated(x, weight, frequencies, positions):
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    half = frequencies.numel()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), positions.double()[:, None] * frequencies.double())[:, None]
    pair = torch.complex(y[..., :half].contiguous(), y[..., half : 2 * half].contiguous()) * turn
    return torch.cat([pair.real, pair.imag, y[..., 2 * half :]], -1)


def _exact_kept(x):
    """What vectors stand for once they are kept in 8 bits."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / 127).clamp(min=LEAST_SCALE)
    return (x / scale).round() * scale


def exact(case, seed):
    """From the definitions in 64 bits, request by request."""
    st = _inputs(case, seed)
    if case["kind"] == "heads":
        return [_exact_rotated(st[n], st[n + "_weight"], st["frequencies"], st["positions"]) for n in ("q", "k")]
    starts = st["starts"].tolist()
    if case["kind"] == "verify":
        tokens, accepted = [], []
        for r, temperature in enumerate(st["temperature"].tolist()):
            begin, end = starts[r], starts[r + 1]
            new = []
            for m in range(begin, end):
                logits = st["logits"][m].double()
                if temperature > 0:
                    p = ((logits - logits.max()) / temperature).exp()
                    p /= p.sum()
                else:
                    p = torch.zeros_like(logits)
                    p[int((logits == logits.max()).nonzero()[0])] = 1.0
                rest = p
                if m < end - 1:
                    t = int(st["tokens"][m + 1])
                    q = st["draft"][m].double() if st["draft"] is not None else (torch.arange(len(p), device=p.device) == t).double()
                    if float(st["uniforms"][m]) * float(q[t]) < float(p[t]):
                        new.append(t)
                        continue
                    rest = (p - q).clamp(min=0)
                    rest = rest if float(rest.sum()) > 0 else p
                total = rest.cumsum(0)
                new.append(int((total <= float(st["uniforms"][end - 1]) * total[-1]).sum()))
                break
            accepted.append(len(new) - 1)
            tokens += new + [-1] * (end - begin - len(new))
        return torch.tensor(tokens, dtype=torch.int32), torch.tensor(accepted, dtype=torch.int32)
    lengths, page, table = st["lengths"].tolist(), case["page"], st["table"].long()
    keys, values = (t.flatten(0, 1) for t in st["history"])
    slots = [(table[r, : -(-n // page)] * page)[:, None].add(torch.arange(page, device="cuda")).flatten()[:n] for r, n in enumerate(lengths)]
    if case["kind"] == "cache":
        position = torch.cat([torch.arange(n - starts[r + 1] + starts[r], n, device="cuda") for r, n in enumerate(lengths)])
        q, k = (_exact_rotated(st[n], st[n + "_weight"], st["frequencies"], position) for n in ("q", "k"))
        written = torch.cat([s[n - starts[r + 1] + starts[r] :] for r, (s, n) in enumerate(zip(slots, lengths))])
        read = torch.cat([s[-min(case["read"], n) :] for s, n in zip(slots, lengths)])
        got = [q]
        for history, x in ((keys, k), (values, st["v"])):
            whole = history.double()
            whole[written] = x.double()
            got.append(_exact_kept(whole[read]))
        return got
    rows, heads, dim = case["rows"], case["kv_heads"], case["dim"]
    got = torch.zeros(rows, case["q_heads"], dim, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lengths):
        k, v = (_exact_kept(t[slots[r]]) for t in (keys, values))
        m = starts[r + 1] - starts[r]
        hidden = torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None]
        for h in range(case["q_heads"]):
            g = h // (case["q_heads"] // heads)
            score = st["q"][starts[r] : starts[r + 1], h].double() @ k[:, g].T / math.sqrt(dim)
            got[starts[r] : starts[r + 1], h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v[:, g]
    return got
