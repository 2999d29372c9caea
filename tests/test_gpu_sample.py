"""splosh_sample against its definition in 64 bits, row by row: filters alone and together, ties, masks,
values that are not finite, and every odd length and layout."""
import math

import numpy as np
import pytest
import torch

from sample_check import check_row, kept_weights, off_borders

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
NAMES = ("temperature", "top_k", "top_p", "min_p")


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def logits_of(rows, vocab, dtype, seed, head=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=gen)
    if head:
        at = torch.randint(0, vocab, (rows, head), generator=gen)
        x.scatter_(1, at, 5.0 + 8.0 * torch.rand(rows, head, generator=gen))
    return x.to(dtype)


def params_of(rows, seed, on=(1, 1, 1, 1), flat=False):
    gen = torch.Generator().manual_seed(seed + 7)

    def rand(low, high):
        return low + (high - low) * torch.rand(rows, generator=gen)

    u, t, p, q = torch.rand(rows, generator=gen), rand(0.4, 1.5), rand(0.3, 0.99), rand(0.01, 0.3)
    k = torch.randint(1, 200, (rows,), generator=gen, dtype=torch.int32)
    pick = torch.rand(4, rows, generator=gen) < 0.6 if on is None else torch.tensor(on).bool()[:, None].expand(4, rows)
    return u, {"temperature": torch.where(pick[0], t, torch.tensor(0.0 if on is None else 1.0)),
               "top_k": torch.where(pick[1], k, torch.tensor(0, dtype=torch.int32)),
               "top_p": torch.where(pick[2], p, torch.tensor(1.0)),
               "min_p": torch.where(pick[3], q, torch.tensor(0.0))}


def call(rt, logits, u, params, **kw):
    dev = {n: None if v is None else v.cuda() for n, v in params.items()}
    tokens, logprobs = rt.sample(logits if logits.is_cuda else logits.cuda(), None if u is None else u.cuda(), **dev, **kw)
    return tokens.cpu(), logprobs.cpu()


def check_all(logits, u, params, tokens, logprobs, label=""):
    for r in range(logits.shape[0]):
        row = {n: float(v[r]) if n != "top_k" else int(v[r]) for n, v in params.items() if v is not None}
        if u is None:
            row["temperature"] = 0.0
        check_row(logits[r].float().cpu().numpy(), tokens[r], float(logprobs[r]), 0.0 if u is None else float(u[r]), **row,
                  label=f"{label} row {r} {row}")


def run(rt, logits, u, params, label=""):
    params = off_borders(logits.float().numpy(), params)
    check_all(logits, u, params, *call(rt, logits, u, params), label)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1025, 4095, 8191, 8192, 8193, 16385, 32003, 100003])
def test_vocabularies(rt, vocab, dtype):
    """Every filter in some rows, at odd and even lengths (fp32: of bf16 logits the sums' borders are
    often ties, which the filters' tests below take one by one)."""
    rows = 12
    logits = logits_of(rows, vocab, torch.float32, vocab, head=min(vocab, 40)).to(dtype)
    u, params = params_of(rows, vocab, None)
    if dtype == torch.bfloat16:
        params["top_p"], params["min_p"] = torch.ones(rows), torch.zeros(rows)
    run(rt, logits, u, params, f"vocab {vocab}")


@pytest.mark.parametrize("on", [(1, 0, 0, 0), (1, 1, 0, 0), (1, 0, 1, 0), (1, 0, 0, 1), (1, 1, 1, 0), (1, 1, 0, 1), (1, 0, 1, 1),
                                (1, 1, 1, 1)])
@pytest.mark.parametrize("head", [0, 40])
def test_filters(rt, on, head):
    """Each filter and each pair, on peaked rows and on flat ones (nuclei of thousands)."""
    rows, vocab = 16, 50021
    u, params = params_of(rows, 3 + sum(on), on)
    run(rt, logits_of(rows, vocab, torch.float32, 5 + head, head), u, params)


@pytest.mark.parametrize("rows", [1, 2, 33, 64, 255, 256, 257, 600])
def test_row_counts(rt, rows):
    u, params = params_of(rows, rows, None)
    run(rt, logits_of(rows, 3001, torch.float32, rows, 30), u, params, f"{rows} rows")


def test_large_vocabulary(rt):
    rows = 6
    u, params = params_of(rows, 11, None)
    run(rt, logits_of(rows, 248320, torch.float32, 12, 48), u, params)
    u, params = params_of(rows, 13, (1, 0, 1, 0))
    run(rt, logits_of(rows, 248320, torch.float32, 14), u, params)


@pytest.mark.parametrize("spread", [1e-4, 0.05, 30.0, 3000.0])
@pytest.mark.parametrize("on", [(1, 1, 0, 0), (1, 0, 1, 0), (1, 1, 1, 1)])
def test_narrow_and_wide_logits(rt, spread, on):
    """Rows whose logits almost agree, and rows where a step of one is thousands."""
    rows = 8
    u, params = params_of(rows, 17, on)
    params["top_k"] *= 10
    run(rt, logits_of(rows, 20011, torch.float32, 18, spread=spread), u, params, f"spread {spread}")


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 0.05, 20.0, 1e6, float("inf")])
def test_temperatures(rt, temperature):
    rows = 6
    logits = logits_of(rows, 9001, torch.float32, 19, 20)
    for on in ((0, 0, 0, 0), (0, 1, 0, 0), (0, 1, 1, 0)):
        u, params = params_of(rows, 20, on)
        params["temperature"] = torch.full((rows,), temperature)
        if temperature == 1e-30:
            params["top_p"] = torch.ones(rows)  # one entry has all the weight: every share ends on it
        run(rt, logits, u, params, f"T {temperature} {on}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5, 700, 9000, 40000])
def test_ties_go_to_the_lowest_index(rt, vocab, dtype):
    """All logits equal: top-k keeps the first k indexes, top-p the first ceil(p n), and u picks among
    them evenly; the greedy row takes index 0."""
    rows = 6
    logits = torch.full((rows, vocab), 1.25, dtype=dtype)
    k = 3
    share = (vocab // 2 + 0.5) / vocab  # half a token past the middle: vocab // 2 + 1 are kept
    u = torch.tensor([0.5, 0.5 / k, 1.0 - 0.5 / k, 0.999, 0.3, 0.5])
    params = {"temperature": torch.tensor([0.0, 1.0, 1.0, 1.0, 2.0, 1.0]),
              "top_k": torch.tensor([0, k, k, 0, 0, vocab + 7], dtype=torch.int32),
              "top_p": torch.tensor([1.0, 1.0, 1.0, share, 1.0, 1.0]),
              "min_p": torch.tensor([0.0, 0.0, 1.0, 0.0, 0.9, 0.0])}
    tokens, logprobs = call(rt, logits, u, params)
    kept = [1, k, k, vocab // 2 + 1, vocab, vocab]
    want = [0] + [int(float(u[r]) * n) for r, n in list(enumerate(kept))[1:]]
    assert tokens.tolist() == want
    assert torch.allclose(logprobs.double(), -torch.tensor(kept).double().log(), rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tied_steps(rt, dtype):
    """A staircase of large groups of equal logits in scattered places: the cut falls inside a group and
    is settled by the index."""
    vocab, groups = 30000, 6
    gen = torch.Generator().manual_seed(23)
    level = torch.randint(0, groups, (vocab,), generator=gen)
    logits = (3.0 - 0.5 * level).to(dtype)[None].repeat(4, 1)
    counts = [int((level == g).sum()) for g in range(groups)]
    k = counts[0] + counts[1] // 2 + 1
    first = torch.cat([(level == 0).nonzero()[:, 0], (level == 1).nonzero()[: k - counts[0], 0]]).sort().values
    w = torch.exp(-0.5 * level.double())[first]
    run_w = w.cumsum(0)
    u = torch.tensor([0.1, 0.4, 0.7, 0.95])
    params = {"temperature": torch.ones(4), "top_k": torch.full((4,), k, dtype=torch.int32), "top_p": torch.ones(4),
              "min_p": torch.zeros(4)}
    tokens, _ = call(rt, logits, u, params)
    assert tokens.tolist() == [int(first[int((run_w <= float(v) * run_w[-1]).sum())]) for v in u]


def test_masks(rt):
    """-inf, the type's lowest value and NaN in masked places; rows that leave one entry or none."""
    vocab = 5000
    for dtype in DTYPES:
        logits = logits_of(8, vocab, torch.float32, 29).to(dtype)
        logits[0] = float("-inf")
        logits[1] = float("nan")
        logits[2, :] = float("-inf")
        logits[2, 4321] = -7.0
        logits[3, ::2] = float("-inf")
        logits[4, 1::2] = float("nan")
        logits[5, 100:] = torch.finfo(dtype).min
        logits[6] = torch.finfo(dtype).min
        logits[7, 17] = logits[7, 4000] = float("inf")
        u = torch.tensor([0.5, 0.5, 0.5, 0.3, 0.9, 0.7, 0.25, 0.6])
        for k, greedy in ((0, False), (3, False), (0, True)):
            params = {"temperature": torch.full((8,), 0.0 if greedy else 0.8), "top_k": torch.full((8,), k, dtype=torch.int32),
                      "top_p": torch.ones(8), "min_p": torch.zeros(8)}
            tokens, logprobs = call(rt, logits, u, params)
            check_all(logits, u, params, tokens, logprobs, f"{dtype} k {k} greedy {greedy}")
            assert tokens[:3].tolist() == [-1, -1, 4321]
            assert tokens[7] == (17 if greedy else 4000)


@pytest.mark.parametrize("dtype", DTYPES)
def test_signalling_nans(rt, dtype):
    """Every kind of NaN (signalling ones too, of both signs) beside the largest logits, in every place of a
    thread's, a wave's and a piece's run: none hides another entry."""
    vocab, rows = 9000, 4
    logits = logits_of(rows, vocab, torch.float32, 61, 20).to(dtype)
    bits = logits.view(torch.int32 if dtype == torch.float32 else torch.int16)
    kinds = ([0x7F800001, 0x7FA00000, 0x7FC00000, -0x7FFFFF, -1] if dtype == torch.float32 else
             [0x7F81, 0x7FA0, 0x7FC0, -0x7F, -1])
    top = torch.topk(logits.float(), 40).indices
    for r in range(rows):
        for i, at in enumerate(top[r].tolist()):
            for step in (-1, 1, 2, 3):
                if 0 <= at + step < vocab and at + step not in set(top[r].tolist()):
                    bits[r, at + step] = kinds[(i + step) % len(kinds)]
    for on in ((1, 1, 0, 0), (1, 0, 1, 0), (1, 0, 0, 1), (1, 0, 0, 0)):
        u, params = params_of(rows, 62, on)
        run(rt, logits, u, params)
    tokens, _ = call(rt, logits, None, {})
    assert torch.equal(tokens.long(), top[:, 0])


def test_parameters_at_their_ends(rt):
    """top_k below 1 and past the vocabulary, top_p of 0, 1 and beyond, min_p of 1 and beyond, u of 0 and
    1 and beyond, and NaN for each."""
    nan, vocab = float("nan"), 3000
    # u, T, k, p, q
    rows = [(0.0, 1, 0, 1.0, 0.0), (1.0, 1, 0, 1.0, 0.0), (-3.0, 1, 0, 1.0, 0.0), (7.0, 1, 9, 1.0, 0.0), (nan, 1, 9, 1.0, 0.0),
            (0.5, 1, -5, 1.0, 0.0), (0.5, 1, 2**31 - 1, 1.0, 0.0), (0.5, 1, 1, 1.0, 0.0), (0.5, 1, 0, 0.0, 0.0),
            (0.5, 1, 0, -1.0, 0.0), (0.5, 1, 0, 2.0, 0.0), (0.5, 1, 0, nan, 0.0), (0.5, 1, 0, 1.0, 1.0), (0.5, 1, 0, 1.0, 3.0),
            (0.5, 1, 0, 1.0, -1.0), (0.5, 1, 0, 1.0, nan), (0.5, nan, 0, 1.0, 0.0), (0.5, -1.0, 0, 1.0, 0.0), (0.9, 0, 50, 0.5, 0.1)]
    logits = logits_of(len(rows), vocab, torch.float32, 31, 20)
    cols = list(zip(*rows))
    u = torch.tensor(cols[0], dtype=torch.float32)
    params = {"temperature": torch.tensor(cols[1], dtype=torch.float32), "top_k": torch.tensor(cols[2], dtype=torch.int32),
              "top_p": torch.tensor(cols[3], dtype=torch.float32), "min_p": torch.tensor(cols[4], dtype=torch.float32)}
    tokens, logprobs = call(rt, logits, u, params)
    check_all(logits, u, params, tokens, logprobs)
    best = logits.argmax(1)
    for r in (7, 8, 9, 12, 13, 16, 17, 18):
        assert tokens[r] == best[r] and logprobs[r] == 0.0, r
    kept = kept_weights(logits[1].numpy())[0]
    assert int(tokens[1]) == int(np.nonzero(kept >= 2.0 ** -40)[0][-1])


@pytest.mark.parametrize("far", [-27.4, -28.5])
def test_a_share_of_weights_below_a_unit(rt, far):
    """One large logit and 200000 that weigh about 2^-40 of it each, 2e-7 to 6e-8 together: with the largest
    p below 1 the share is not reached before them. The token is the large one's for every u from 1e-6 to 1 - 1e-6."""
    rows, vocab = 8, 200003
    logits = (far + 0.01 * torch.rand(rows, vocab, generator=torch.Generator().manual_seed(63))).float()
    at = torch.arange(rows) * 23456 + 7
    logits[torch.arange(rows), at] = 0.0
    u = torch.linspace(1e-6, 1.0 - 1e-6, rows)
    top_p = torch.full((rows,), 1.0 - 2.0 ** -24)
    for params in ({"top_p": top_p}, {"top_p": top_p, "min_p": torch.full((rows,), 0.01)},
                   {"top_p": top_p, "top_k": torch.full((rows,), 5000, dtype=torch.int32)}):
        tokens, logprobs = call(rt, logits, u, params)
        assert torch.equal(tokens.long(), at) and (logprobs <= 0).all() and (logprobs >= -1e-6).all()


@pytest.mark.parametrize("offset", [0.0, -3.0, 3.0])
def test_temperatures_below_the_normal_numbers(rt, offset):
    """The largest entry alone has weight; of two equal ones each half of it."""
    rows, vocab = 4, 9001
    logits = -1.0 - torch.rand(rows, vocab, generator=torch.Generator().manual_seed(64)) + offset
    logits[:, [700, 8800]] = offset
    u = torch.tensor([0.0, 0.49, 0.51, 1.0])
    for t in (2.0 ** -149, 1e-40, 2.0 ** -126):
        for params in ({}, {"top_p": torch.full((rows,), 0.9)}, {"min_p": torch.full((rows,), 0.5)},
                       {"top_k": torch.full((rows,), 50, dtype=torch.int32)}):
            tokens, logprobs = call(rt, logits, u, {"temperature": torch.full((rows,), t), **params})
            assert tokens.tolist() == [700, 700, 8800, 8800]
            assert (logprobs + math.log(2.0)).abs().max() <= 2.0 ** -20


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 1e36, 3e38, float("inf")])
def test_masks_at_the_largest_temperatures(rt, temperature, dtype):
    """NaN and -inf weigh nothing where every other weight is the same, too."""
    rows, vocab = 6, 20011
    logits = logits_of(rows, vocab, torch.float32, 65).to(dtype)
    mask = torch.rand(rows, vocab, generator=torch.Generator().manual_seed(66))
    logits[mask < 0.5] = -math.inf
    logits[mask < 0.1] = math.nan
    for on in ((0, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 1, 0)):
        u, params = params_of(rows, 67, on)
        params["temperature"] = torch.full((rows,), temperature)
        run(rt, logits, u, params, f"{on}")


@pytest.mark.parametrize("scale", [2.0 ** 100, 2.0 ** 112, 2.0 ** 120])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_logits_of_the_largest_sizes(rt, scale, sign):
    """At both ends of fp32, where a bin is 2^-6 of a logit and the lowest bins are those of NaN and -inf."""
    rows, vocab = 6, 9001
    gen = torch.Generator().manual_seed(68)
    logits = sign * scale * (1.0 + torch.rand(rows, vocab, generator=gen))
    logits[torch.rand(rows, vocab, generator=gen) < 0.3] = -math.inf
    logits[torch.rand(rows, vocab, generator=gen) < 0.1] = math.nan
    for on in ((0, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 1, 1, 1)):
        u, params = params_of(rows, 69, on)
        params["temperature"] = torch.full((rows,), scale / 8)
        run(rt, logits, u, params, f"{on}")


@pytest.mark.parametrize("vocab,dtype", [(524287, torch.float32), (600001, torch.bfloat16), (1 << 21, torch.float32),
                                         (1 << 21, torch.bfloat16)])
def test_largest_vocabularies(rt, vocab, dtype):
    """More strips than a workgroup has threads; bf16's ties overflow the list, and the row is searched whole."""
    rows = 2
    logits = logits_of(rows, vocab, torch.float32, vocab, 48).to(dtype)
    wide = torch.full((rows, vocab + 3), 1e4, dtype=dtype)
    wide[:, 1 : 1 + vocab] = logits
    for on in ((1, 0, 0, 0), (1, 1, 0, 1), (1, 0, 1, 0)):
        u, params = params_of(rows, vocab + 1, on)
        params = off_borders(logits.float().numpy(), params)
        check_all(logits, u, params, *call(rt, wide.cuda()[:, 1 : 1 + vocab], u, params), f"{on}")


def test_defaults(rt):
    """No uniforms: greedy. No parameters: temperature 1 and no filter."""
    logits = logits_of(9, 2500, torch.float32, 37)
    tokens, logprobs = call(rt, logits, None, {})
    assert torch.equal(tokens.long(), logits.argmax(1)) and not logprobs.any()
    u = torch.rand(9, generator=torch.Generator().manual_seed(38))
    run(rt, logits, u, {})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,pad", [(1000, 1), (1000, 3), (4099, 2), (20000, 8)])
def test_strides(rt, vocab, pad, dtype):
    """Rows of a wider buffer at odd places; what surrounds them (larger than any logit) is not looked at."""
    rows = 10
    logits = logits_of(rows, vocab, torch.float32, vocab, 30).to(dtype)
    wide = torch.full((rows, vocab + 2 * pad), 1e4, dtype=dtype, device="cuda")
    wide[:, pad:-pad] = logits.cuda()
    u, params = params_of(rows, vocab, (1, 1, 0, 0))
    check_all(logits, u, params, *call(rt, wide[:, pad:-pad], u, params))


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_rows(rt, dtype):
    """Rows that begin past 2^32 bytes."""
    size = torch.finfo(dtype).bits // 8
    stride = (1 << 32) // size // 3 + 5
    wide = torch.zeros(4 * stride + 2000, dtype=dtype, device="cuda")
    logits = logits_of(5, 2000, torch.float32, 41, 10).to(dtype)
    view = wide.as_strided((5, 2000), (stride, 1))
    view.copy_(logits.cuda())
    u, params = params_of(5, 42, (1, 1, 0, 0))
    check_all(logits, u, params, *call(rt, view, u, params))


def test_repeatable_and_workspace_returned_clean(rt):
    """The same answer every time, on one workspace that calls of other shapes share; its counters are
    zero after each."""
    rows, vocab = 40, 30011
    ws = torch.zeros(max(rt.sample_workspace_bytes(rows, vocab), rt.sample_workspace_bytes(300, 2000)), dtype=torch.uint8,
                     device="cuda")
    logits = logits_of(rows, vocab, torch.float32, 43, 40).cuda()
    u, params = params_of(rows, 44, None)
    first = call(rt, logits, u, params)
    other = logits_of(300, 2000, torch.bfloat16, 45).cuda()
    ou, oparams = params_of(300, 46, None)
    for _ in range(3):
        got = call(rt, logits, u, params, workspace=ws)
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
        call(rt, other, ou, oparams, workspace=ws)
        assert not ws[: rt.WORKSPACE_COUNTER_BYTES].any()


def test_rows_do_not_depend_on_each_other(rt):
    rows, vocab = 20, 12345
    logits = logits_of(rows, vocab, torch.float32, 47, 40).cuda()
    u, params = params_of(rows, 48, None)
    tokens, logprobs = call(rt, logits, u, params)
    for r in (0, 7, 19):
        one = call(rt, logits[r : r + 1], u[r : r + 1], {n: v[r : r + 1] for n, v in params.items()})
        assert one[0][0] == tokens[r] and one[1][0] == logprobs[r]


def test_outputs_past_the_last_row_stay(rt):
    rows = 5
    logits = logits_of(rows, 900, torch.float32, 49)
    out = torch.full((8,), 77, dtype=torch.int32, device="cuda")
    lp = torch.full((8,), 77.0, device="cuda")
    rt.sample(logits.cuda(), torch.full((8,), 0.5, device="cuda"), out=out, logprobs=lp)
    assert (out[rows:] == 77).all() and (lp[rows:] == 77.0).all() and (lp[:rows] < 0).all()


def test_streams(rt):
    """Two calls at once, each on a stream and a workspace of its own."""
    cases = []
    for s in (51, 52):
        logits = logits_of(16, 60000, torch.float32, s, 40)
        u, params = params_of(16, s, None)
        params = off_borders(logits.numpy(), params)
        cases.append((logits, u, params, logits.cuda(), u.cuda(), {n: v.cuda() for n, v in params.items()}, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [rt.sample(c[3], c[4], **c[5], stream=c[6]) for c in cases for _ in range(3)]
    torch.cuda.synchronize()
    for i, (tokens, logprobs) in enumerate(got):
        check_all(*cases[i // 3][:3], tokens.cpu(), logprobs.cpu())


def test_graph_replays(rt):
    """Captured, then replayed with other logits and parameters written into the same tensors."""
    rows, vocab = 12, 40009
    logits = logits_of(rows, vocab, torch.float32, 53, 40).cuda()
    u, params = params_of(rows, 54, None)
    dev = {"uniforms": u.cuda(), **{n: v.cuda() for n, v in params.items()}}
    ws = torch.zeros(rt.sample_workspace_bytes(rows, vocab), dtype=torch.uint8, device="cuda")
    out, lp = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, device="cuda")
    rt.sample(logits, **dev, out=out, logprobs=lp, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.sample(logits, **dev, out=out, logprobs=lp, workspace=ws)
    for seed in range(55, 59):
        fresh = logits_of(rows, vocab, torch.float32, seed, 40)
        u, params = params_of(rows, seed, None)
        params = off_borders(fresh.numpy(), params)
        logits.copy_(fresh)
        dev["uniforms"].copy_(u)
        for n, v in params.items():
            dev[n].copy_(v)
        eager = rt.sample(logits, **dev)
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lp, eager[1])
        check_all(fresh, u, params, out.cpu(), lp.cpu())


def test_draws_follow_the_distribution(rt):
    """65536 evenly spaced draws of one row: each token as often as its weight says, to a draw."""
    logits = torch.randn(1, 40, generator=torch.Generator().manual_seed(59))
    n = 65536
    u = (torch.arange(n) + 0.5) / n
    tokens, _ = call(rt, logits.expand(n, 40).contiguous(), u, {"top_k": torch.full((n,), 25, dtype=torch.int32)})
    w, _ = kept_weights(logits[0].numpy(), top_k=25)
    count = np.bincount(tokens.numpy(), minlength=40)
    assert np.abs(count - n * w / w.sum()).max() <= 1.0 + 1e-3


def test_python_refusals(rt):
    from splosh_amd._lib import SploshError
    logits = torch.randn(4, 100).cuda()
    u = torch.rand(4).cuda()

    def refused(case, *args, **kw):
        with pytest.raises(SploshError) as e:
            rt.sample(*args, **kw)
        assert e.value.case == case, e.value

    refused("unsupported", logits[0], u)
    refused("unsupported", logits.t(), u)
    refused("unsupported", logits.half(), u)
    refused("unsupported", logits, u.double())
    refused("unsupported", logits, u.cpu())
    refused("bufferTooSmall", logits, u[:3])
    refused("unsupported", logits, u, top_k=u)
    refused("unsupported", logits, u, temperature=u[:, None])
    refused("unsupported", logits, u, out=torch.zeros(4, dtype=torch.int64, device="cuda"))
    refused("bufferTooSmall", logits, u, out=torch.zeros(3, dtype=torch.int32, device="cuda"))
    refused("invalidShape", logits[:0], u)
    refused("workspaceTooSmall", logits, u, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    refused("nullPointer", logits.cpu(), u)
