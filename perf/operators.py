"""The measured work of a packed step's per-request operators: what the rows of one batched
projection do not share.

Kinds of case, each one pass through one operator:

* ``adapters`` -- low-rank adapters beside shared projections of one activation: row m of each
  output gains scale_s * b_s (a_s x[m]) of its request's adapter s, in place; rows without an
  adapter stay as they are. One projection, or several of the same activation (q/k/v, gate/up).
* ``sample`` -- the next token of every row from the lm_head's logits: temperature, top-k, top-p
  and min-p, each row with its own, from given uniform random numbers, and the logarithm of the
  probability that the token was drawn with.

Sizes are those of the library's benchmark workloads (hidden 5120, MLP 17408, vocabulary 248320)
and odd ones of the same form. With ``own`` false the operators are computed with elementary torch
operations, with ``own`` true by the library's entry points.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    def adapters(name, rows, hidden, outputs, rank, slots, spread, dtype, mixed=False, padded=False):
        return {"name": name, "kind": "adapters", "rows": rows, "hidden": hidden, "outputs": outputs, "rank": rank,
                "slots": slots, "spread": spread, "dtype": dtype, "mixed": mixed, "padded": padded}

    def sample(name, rows, vocab, dtype, params, flat=False, padded=False):
        return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "params": params,
                "flat": flat, "padded": padded}

    return [
        # One token of one request: all latency.
        adapters("adapters_decode_1", 1, 5120, "5120", 16, 4, "rows", "bf16"),
        # Eight requests of one token each, an adapter each, on q, k and v at once.
        adapters("adapters_qkv_8", 8, 5120, "5120,1024,1024", 16, 8, "rows", "bf16"),
        # Eight sessions of eight drafted tokens, gate and up at once in fp32 (silu * up reads fp32).
        adapters("adapters_gate_up_64", 64, 5120, "17408,17408", 16, 8, "requests", "f32"),
        # Sixty-four requests on thirty-two adapters of different ranks, the down projection onto
        # the fp32 residual.
        adapters("adapters_down_64", 64, 17408, "5120", 64, 32, "rows", "f32", mixed=True),
        # An odd batch of an odd projection, rows of wider buffers, a rank that is no power of two.
        adapters("adapters_odd_37", 37, 1001, "777", 12, 5, "rows", "bf16", padded=True),
        # Three prompts together, and a whole prefill step of four.
        adapters("adapters_prompt_333", 333, 6144, "5120", 64, 3, "requests", "f32"),
        adapters("adapters_prefill_2048", 2048, 5120, "17408", 16, 4, "requests", "bf16"),
        # One token's logits with every filter on.
        sample("sample_1", 1, 248320, "f32", "filters"),
        # A verify step of 64 rows whose requests ask for different things: greedy, temperature
        # alone, top-k, top-p, min-p and all of them.
        sample("sample_verify_64", 64, 248320, "f32", "mixed"),
        # The same rows from bf16 logits with the temperature alone: no cut to find.
        sample("sample_temperature_64", 64, 248320, "bf16", "temperature"),
        # Nuclei of thousands of tokens: flat bf16 logits, full of ties, of an odd vocabulary.
        sample("sample_nucleus_16", 16, 100003, "bf16", "top_p", flat=True, padded=True),
        # A wide batch on a small odd vocabulary.
        sample("sample_batch_256", 256, 32003, "f32", "mixed"),
    ]


def _between(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _between(rng, 1000, 248320)
        rows = min(_between(rng, 1, 256), 64 * 248320 // vocab)
        return {"kind": "sample", "rows": rows, "vocab": vocab, "dtype": rng.choice(["f32", "bf16"]),
                "params": rng.choice(["filters", "mixed", "mixed", "temperature", "top_p", "top_k", "min_p", "greedy"]),
                "flat": rng.random() < 0.3, "padded": rng.random() < 0.3}
    rows = rng.choice([1, rng.randint(2, 16), rng.randint(17, 64), rng.randint(65, 256), _between(rng, 257, 2048)])
    step = rng.choice([1, 8, 64, 128])  # odd sizes, and those of real projections
    hidden = max(step, _between(rng, 512, 17408) // step * step)
    count = rng.choice([1, 1, 2, 3])
    most = 17408 if rows <= 64 else max(256, min(17408, 2048 * 17408 // rows // count // 2))
    outputs = ",".join(str(max(step, _between(rng, 256, most) // step * step)) for _ in range(count))
    rank = rng.choice([4, 8, 16, 16, 32, 64, 128, rng.randint(1, 128)])
    spread = "rows" if rows <= 64 and rng.random() < 0.6 else "requests"
    slots = rng.randint(1, max(1, min(32, (1024 if rows <= 64 else 256) // rank)))
    return {"kind": "adapters", "rows": rows, "hidden": hidden, "outputs": outputs, "rank": rank, "slots": slots,
            "spread": spread, "dtype": rng.choice(["f32", "bf16"]), "mixed": rng.random() < 0.3,
            "padded": rng.random() < 0.3}


# ---- inputs, from the seed alone ----------------------------------------------------------------


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed(seed * 1000 + salt)


def _rows_of(t, padded):
    """`t` as rows of a wider buffer, where the case asks for that."""
    if not padded:
        return t
    wide = torch.zeros(t.shape[0], t.shape[1] + 24, dtype=t.dtype, device=t.device)
    wide[:, : t.shape[1]] = t
    return wide[:, : t.shape[1]]


def _outputs(case):
    return [int(n) for n in case["outputs"].split(",")]


def _slots_of(case, seed):
    """The adapter of each row: -1 for none. `rows`: every row a request of its own. `requests`:
    runs of rows of one request, of uneven lengths."""
    rows, slots, gen = case["rows"], case["slots"], _gen(seed, 1)
    if case["spread"] == "rows":
        low = -1 if rows > 1 else 0
        return torch.randint(low, slots, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    requests = min(rows, slots)
    order = torch.randperm(slots, device="cuda", generator=gen)[:requests].to(torch.int32)
    starts = torch.randperm(rows - 1, device="cuda", generator=gen)[: requests - 1] + 1 if rows > 1 else None
    marks = torch.zeros(rows, dtype=torch.int64, device="cuda")
    if starts is not None:
        marks[starts] = 1
    return order[marks.cumsum(0)]


def _ranks_of(case, seed):
    """The rank of each adapter: all the same, or some of them shorter (an adapter of rank 0 is one
    that leaves the projection alone)."""
    full = torch.full((case["slots"],), case["rank"], dtype=torch.int32, device="cuda")
    if not case["mixed"]:
        return full
    shift = torch.randint(0, 4, (case["slots"],), dtype=torch.int32, device="cuda", generator=_gen(seed, 2))
    return full >> shift


def _adapter_inputs(case, seed):
    rows, hidden, rank, slots = case["rows"], case["hidden"], case["rank"], case["slots"]
    gen = _gen(seed, 3)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    x = _rows_of(normal(rows, hidden).to(torch.bfloat16), case["padded"])
    a = [(normal(slots, rank, hidden) / math.sqrt(hidden)).to(torch.bfloat16) for _ in _outputs(case)]
    b = [(normal(slots, n, rank) * 0.05).to(torch.bfloat16) for n in _outputs(case)]
    scales = 0.5 + 1.5 * torch.rand(slots, device="cuda", generator=gen)
    outs = [_rows_of(normal(rows, n).to(DTYPES[case["dtype"]]), case["padded"]) for n in _outputs(case)]
    return {"x": x, "a": a, "b": b, "scales": scales, "ranks": _ranks_of(case, seed), "outs": outs,
            "slots": _slots_of(case, seed)}


def _logits(case, seed):
    """A bulk of unlikely tokens and, unless `flat`, a head of a few dozen likely ones that decays."""
    rows, vocab = case["rows"], case["vocab"]
    gen = _gen(seed, 4)
    logits = 2.0 * torch.randn(rows, vocab, device="cuda", generator=gen)
    if not case["flat"]:
        head = min(vocab, 48)
        at = torch.randint(0, vocab, (rows, head), device="cuda", generator=gen)
        bonus = 14.0 - 8.0 * torch.rand(rows, head, device="cuda", generator=gen).sqrt()
        logits.scatter_reduce_(1, at, bonus, "amax")  # (a place drawn twice: the larger, whatever the order)
    return _rows_of(logits.to(DTYPES[case["dtype"]]), case["padded"])


def _sample_inputs(case, seed):
    rows, gen = case["rows"], _gen(seed, 5)

    def rand(low, high):
        return low + (high - low) * torch.rand(rows, device="cuda", generator=gen)

    temperature, top_p, min_p = rand(0.5, 1.3), rand(0.7, 0.98), rand(0.02, 0.2)
    top_k = torch.randint(5, 101, (rows,), dtype=torch.int32, device="cuda", generator=gen)
    on = {"filters": (1, 1, 1, 1), "temperature": (1, 0, 0, 0), "top_p": (1, 0, 1, 0), "top_k": (1, 1, 0, 0),
          "min_p": (1, 0, 0, 1), "greedy": (0, 0, 0, 0)}.get(case["params"])
    if on is None:  # every row its own choice of them
        on = torch.rand(4, rows, device="cuda", generator=gen) < torch.tensor([[0.85], [0.4], [0.4], [0.3]], device="cuda")
    else:
        on = torch.tensor(on, device="cuda").bool()[:, None].expand(4, rows)
    zero = torch.zeros_like(temperature)
    return {"logits": _logits(case, seed), "uniforms": torch.rand(rows, device="cuda", generator=gen),
            "temperature": torch.where(on[0], temperature, zero), "top_k": torch.where(on[1], top_k, torch.zeros_like(top_k)),
            "top_p": torch.where(on[2], top_p, zero + 1.0), "min_p": torch.where(on[3], min_p, zero)}


def prepare(case, seed):
    kind = case["kind"]
    st = _adapter_inputs(case, seed) if kind == "adapters" else _sample_inputs(case, seed)
    st["kind"] = kind
    if own:  # the handles, outputs and scratch that a serving program keeps between steps
        from splosh_amd import runtime as rt
        if kind == "adapters":
            st["adapters"] = [rt.Adapters(a, b, st["scales"], st["ranks"]) for a, b in zip(st["a"], st["b"])]
            need = rt.adapters_workspace_bytes(st["adapters"], case["rows"])
        else:
            rows = case["rows"]
            st["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
            st["logprobs"] = torch.empty(rows, dtype=torch.float32, device="cuda")
            need = rt.sample_workspace_bytes(rows, case["vocab"])
        st["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    return st


# ---- the operators ------------------------------------------------------------------------------


def _plain_adapters(st):
    """All adapters' products of all rows, of which each row keeps its own adapter's ranks."""
    slots, ranks = st["slots"], st["ranks"]
    count, rank = st["a"][0].shape[:2]
    at = torch.arange(count * rank, device=slots.device)
    keep = (slots[:, None] == at // rank) & (at % rank < ranks[at // rank])
    factor = torch.where(keep, st["scales"][at // rank], 0.0)
    x = st["x"].float()

    def add(out, a, b):
        low = (x @ a.float().reshape(count * rank, -1).T) * factor
        return out.copy_(out.float() + low @ b.float().transpose(1, 2).reshape(count * rank, -1))

    return [add(*p) for p in zip(st["outs"], st["a"], st["b"])]


def _plain_sample(st):
    """By sorting each row, in 64 bits: the sums decide between neighbouring tokens."""
    logits = st["logits"].double()
    greedy = st["temperature"] <= 0
    scaled = logits / torch.where(greedy, 1.0, st["temperature"]).double()[:, None]
    values, order = torch.sort(scaled, dim=1, descending=True, stable=True)
    weight = torch.exp(values - values[:, :1])
    place = torch.arange(weight.shape[1], device=weight.device)
    top_k = torch.where(st["top_k"] > 0, st["top_k"], weight.shape[1])
    top_k = torch.where(greedy, 1, top_k)
    kept = torch.where(place < top_k[:, None], weight, 0.0)
    total = kept.cumsum(1)
    before = total - kept
    inside = (before < st["top_p"].double()[:, None] * total[:, -1:]) | (st["top_p"] >= 1)[:, None] | (place == 0)
    inside &= weight >= st["min_p"].double().clamp(max=1.0)[:, None]
    kept = torch.where(inside, kept, 0.0)
    # Back in the order of the vocabulary, the first token whose running sum passes the draw.
    kept = torch.zeros_like(kept).scatter_(1, order, kept)
    total = kept.cumsum(1)
    passed = total > st["uniforms"].double()[:, None] * total[:, -1:]
    token = passed.to(torch.uint8).argmax(1, keepdim=True)
    return token[:, 0].int(), torch.log(kept.gather(1, token) / total[:, -1:])[:, 0].float()


def run(st):
    if own:
        from splosh_amd import runtime as rt
        if st["kind"] == "adapters":
            return rt.add_adapters_group(st["outs"], st["x"], st["adapters"], st["slots"], workspace=st["workspace"])
        return rt.sample(st["logits"], st["uniforms"], st["temperature"], st["top_k"], st["top_p"], st["min_p"],
                         out=st["tokens"], logprobs=st["logprobs"], workspace=st["workspace"])
    return _plain_adapters(st) if st["kind"] == "adapters" else _plain_sample(st)


# ---- what a pass cannot do without, and what it has to give ---------------------------------------


def work(case):
    rows = case["rows"]
    if case["kind"] == "sample":
        size = 4 if case["dtype"] == "f32" else 2
        values = rows * case["vocab"]
        return {"bytes": values * size + rows * 28, "flops": 3 * values}
    hidden, slots, rank = case["hidden"], case["slots"], case["rank"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["mixed"]:  # the mean of the ranks
        rank = sum(rank >> s for s in range(4)) / 4
    if case["spread"] == "rows":  # one value of slots + 1 says "none"; the adapters that the rows reach
        values = slots + (rows > 1)
        with_one = rows * slots / values
        used = slots * (1 - (1 - 1 / values) ** rows)
    else:
        with_one, used = rows, min(rows, slots)
    outputs = _outputs(case)
    read = with_one * hidden * 2 + used * rank * (len(outputs) * hidden + sum(outputs)) * 2 + rows * 4
    return {"bytes": read + 2 * with_one * sum(outputs) * size,
            "flops": 2 * with_one * rank * (len(outputs) * hidden + sum(outputs))}


def exact(case, seed):
    """From the definitions in 64 bits: adapter by adapter, and row by row."""
    if case["kind"] == "adapters":
        st = _adapter_inputs(case, seed)
        got = [out.double().clone() for out in st["outs"]]
        for s in range(case["slots"]):
            mine, rank = st["slots"] == s, int(st["ranks"][s])
            for out, a, b in zip(got, st["a"], st["b"]):
                low = st["x"][mine].double() @ a[s, :rank].double().T
                out[mine] += st["scales"][s].double() * (low @ b[s, :, :rank].double().T)
        return got
    st = _sample_inputs(case, seed)
    tokens, logprobs = [], []
    params = zip(*(st[n].tolist() for n in ("uniforms", "temperature", "top_k", "top_p", "min_p")))
    for logits, (u, temperature, top_k, top_p, min_p) in zip(st["logits"], params):
        logits = logits.double()
        if temperature <= 0:
            tokens.append(int((logits == logits.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        order = torch.sort(-logits, stable=True).indices
        weight = ((logits[order] - logits.max()) / temperature).exp()
        if top_k > 0:
            order, weight = order[:top_k], weight[:top_k]
        if top_p < 1:
            n = 1 + int((weight.cumsum(0) < top_p * weight.sum()).sum())
            order, weight = order[:n], weight[:n]
        if min_p > 0:
            order, weight = order[weight >= min_p], weight[weight >= min_p]
        order, by_index = order.sort()
        weight = weight[by_index]
        at = int((weight.cumsum(0) <= u * weight.sum()).sum())
        tokens.append(int(order[at]))
        logprobs.append(float((weight[at] / weight.sum()).log()))
    return (torch.tensor(tokens, dtype=torch.int32), torch.tensor(logprobs, dtype=torch.float64))
