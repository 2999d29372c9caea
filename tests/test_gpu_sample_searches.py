"""splosh_sample where a row's cut is searched for in a long list or in the whole row, against its definition in
64 bits."""
import math

import numpy as np
import pytest
import torch

from sample_check import off_borders
from test_gpu_sample import call, check_all, logits_of, params_of, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


@pytest.mark.parametrize("k,vocab,spread", [(65, 20011, 2.0), (150, 50021, 2.0), (600, 50021, 1.0), (600, 248320, 2.0),
                                            (600, 9001, 0.0), (9000, 30011, 2.0)])
def test_top_k_and_top_p_of_long_lists(rt, k, vocab, spread):
    """Both cuts, one after the other, from more than 64 keys, or (equal logits, and more than 8192 keys between
    the two cuts) from the whole row: the second search starts from the first one's results in every wave. The same
    tokens and logprobs every time."""
    rows = 48
    logits = logits_of(rows, vocab, torch.float32, k, spread=spread)
    u, params = params_of(rows, k, (1, 1, 1, 0))
    params["top_k"] = k - torch.arange(rows, dtype=torch.int32) % 7
    params = off_borders(logits.numpy(), params)
    dev = logits.cuda()
    first = call(rt, dev, u, params)
    check_all(logits, u, params, *first)
    for _ in range(8):
        tokens, logprobs = call(rt, dev, u, params)
        assert torch.equal(tokens, first[0]) and torch.equal(logprobs, first[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_stretches_weigh_nothing_at_the_largest_temperatures(rt, dtype):
    """Stretches of -inf and NaN before the first entry that can be chosen, temperatures at which a weight far below
    the largest is still a fraction of it: the draws of 0 and just above take the first entry that can be chosen."""
    rows, vocab, first = 96, 9001, 3100
    logits = logits_of(rows, vocab, torch.float32, 71).to(dtype)
    logits[:, :first] = -math.inf
    logits[:, 40:2000:3] = math.nan
    logits[:, first + 20:] = -math.inf
    u = torch.zeros(rows)
    u[1::2] = 1e-9
    params = {"temperature": torch.tensor(np.geomspace(4e36, 3.3e38, rows).astype(np.float32)),
              "top_k": torch.zeros(rows, dtype=torch.int32), "top_p": torch.ones(rows), "min_p": torch.zeros(rows)}
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    tokens, logprobs = call(rt, logits, u, params, out=out)
    assert tokens.tolist() == [first] * rows
    check_all(logits, u, params, tokens, logprobs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_length_of_a_short_list(rt, dtype):
    """Lists of 1 to 64 keys, ranked at once: k of them kept, and of these a share that ends at each place in turn,
    between the sums before and after it."""
    rows, vocab = 64, 9001
    gen = torch.Generator().manual_seed(73)
    logits = (-40.0 - torch.rand(rows, vocab, generator=gen)).to(dtype)
    steps = (-0.0625 * torch.arange(rows)).to(dtype)  # (weights 6% apart)
    for r in range(rows):
        logits[r, torch.randperm(vocab, generator=gen)[:rows]] = steps
    w = torch.exp(steps.double())
    for shift in (0, 5, 40):
        k = torch.arange(1, rows + 1)
        ends = (k * 7 + shift) % k  # place of the last that the share keeps
        run = torch.stack([w.cumsum(0)[e] for e in ends])
        share = (run - 0.5 * w[ends]) / w.cumsum(0)[k - 1]
        u = torch.rand(rows, generator=gen)
        params = {"temperature": torch.ones(rows), "top_k": k.int(), "top_p": share.float(), "min_p": torch.zeros(rows)}
        params["top_k"][::3] += 2  # (the cut past the share, and where the list is longer than k)
        params = off_borders(logits.float().numpy(), params)
        check_all(logits, u, params, *call(rt, logits, u, params), f"shift {shift}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [777, 12345, 40009])
def test_the_same_row_at_every_alignment(rt, vocab, dtype):
    """A row's token and the bits of its logprob do not depend on where the row begins."""
    rows = 300
    logits = logits_of(rows, vocab, torch.float32, 77, head=20, spread=3.0).to(dtype)
    for on in ((1, 0, 0, 0), (1, 0, 1, 0), (1, 1, 1, 0), (1, 0, 0, 1), None):
        u, params = params_of(rows, 78, on)
        want = call(rt, logits, u, params)
        places = 16 // dtype.itemsize
        for at in range(places):
            # (A stride of whole 16 bytes: every row begins at the same place in its 16 bytes.)
            wide = torch.full((rows, (vocab + 2 * places) // places * places), 1e4, dtype=dtype, device="cuda")
            wide[:, at : at + vocab] = logits.cuda()
            got = call(rt, wide[:, at : at + vocab], u, params)
            off = (got[0] != want[0]) | (got[1].view(torch.int32) != want[1].view(torch.int32))
            assert int(off.sum()) == 0, f"{on} at {at}"


@pytest.mark.parametrize("offset", [-300.0, -20.0, 15.0, 30.0, 100.0, 4000.0])
def test_logits_about_another_value(rt, offset):
    """A common offset: the bins about it are wider, the lists longer, and from some offset on rows are searched whole."""
    rows, vocab = 8, 100003
    logits = logits_of(rows, vocab, torch.float32, 79) + offset
    for on in ((1, 0, 1, 0), (1, 1, 1, 0), (1, 0, 1, 1)):
        u, params = params_of(rows, 80, on)
        run(rt, logits, u, params, f"{offset} {on}")


@pytest.mark.parametrize("head", [0, 40])
@pytest.mark.parametrize("top_p", [0.9995, 0.9999, 0.99999, 1.0 - 2.0 ** -24])
def test_shares_next_to_the_whole(rt, top_p, head):
    """Shares that the bins cannot tell from the whole weight."""
    rows, vocab = 8, 60013
    logits = logits_of(rows, vocab, torch.float32, 81, head)
    u, params = params_of(rows, 82, (1, 0, 1, 0))
    params["top_p"] = torch.full((rows,), top_p)
    run(rt, logits, u, params)
    params["top_k"] = torch.full((rows,), 20000, dtype=torch.int32)
    run(rt, logits, u, params)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("far", [-16.0, -22.0, -25.0])
def test_logprobs_of_unlikely_tokens(rt, far, dtype):
    """One large logit and 100000 of about e^far of its weight: a draw from among those has its own logprob, to fp32's
    last places of it and 2^-20 for the whole weight."""
    rows, vocab = 16, 100003
    gen = torch.Generator().manual_seed(83)
    logits = (far + 0.5 * torch.rand(rows, vocab, generator=gen)).to(dtype)
    logits[:, 0] = 0.0
    u = torch.full((rows,), 1.0 - 2.0 ** -22)
    for params in ({}, {"min_p": torch.full((rows,), 2.0 ** -39)}, {"top_k": torch.full((rows,), 99000, dtype=torch.int32)}):
        tokens, logprobs = call(rt, logits, u, params)
        z = torch.gather(logits.double(), 1, tokens.long()[:, None])[:, 0]
        kept = logits.double().exp() if "top_k" not in params else torch.topk(logits.double(), 99000).values.exp()
        want = z - kept.sum(1).log()
        assert (tokens > 0).all() and (z <= far + 0.5).all()
        assert ((logprobs.double() - want).abs() <= 2.0 ** -20 + 2.0 ** -23 * want.abs()).all(), (logprobs.double() - want).abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-30, 0.7, 1e38, math.inf])
def test_infinite_entries_with_every_filter(rt, temperature, dtype):
    """+inf among the entries: those alone have weight, whatever filter they pass, in one piece or in several."""
    rows, vocab = 6, 20011
    logits = logits_of(rows, vocab, torch.float32, 84).to(dtype)
    for r in range(rows):
        logits[r, torch.randperm(vocab, generator=torch.Generator().manual_seed(r))[: 1 + 29 * r]] = math.inf
    logits[:, 100:4000:3] = -math.inf
    for on in ((1, 0, 0, 0), (1, 1, 0, 0), (1, 0, 1, 0), (1, 0, 0, 1), (1, 1, 1, 0), (1, 0, 1, 1), (1, 1, 1, 1)):
        u, params = params_of(rows, 85, on)
        params["temperature"] = torch.full((rows,), temperature)
        run(rt, logits, u, params, f"{on}")
