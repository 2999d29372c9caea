"""splosh_verify against its definition in 64 bits, request by request."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def weights(logits, temperature):
    """p in 64 bits, zeros for a row without entries."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.max()
    if top == -math.inf:
        return torch.zeros_like(x)
    if not temperature > 0:
        p = torch.zeros_like(x)
        p[int((x == top).nonzero()[0])] = 1.0
        return p
    w = (x == math.inf).double() if top == math.inf else ((x - top) / max(temperature, 2.0 ** -126)).exp()
    return w / w.sum()


def verified(logits, tokens, u, temperature, draft):
    """(tokens, accepted, how near the nearest decision was) of one request."""
    n, vocab = logits.shape
    got, margin = [], math.inf
    u = [max(x, 0.0) if x == x else 0.0 for x in u]
    for j in range(n):
        p = weights(logits[j], temperature)
        rest = p
        if j < n - 1:
            t = int(tokens[j + 1])
            q = draft[j].double() if draft is not None else (torch.arange(vocab) == t).double()
            if 0 <= t < vocab:
                margin = min(margin, abs(u[j] * float(q[t]) - float(p[t])))
                if u[j] * float(q[t]) < float(p[t]):
                    got.append(t)
                    continue
            rest = torch.where(torch.isnan(q), 0.0, (p - q).clamp(min=0))
            rest = rest if float(rest.sum()) > 0 else p
        running = rest.cumsum(0)
        total = float(running[-1])
        if total == 0:
            got.append(-1)
            break
        draw = u[-1] * total
        passed = (running > draw) & (rest > 0)
        token = int(passed.nonzero()[0]) if passed.any() else int((rest > 0).nonzero()[-1])
        if u[-1] < 1:
            margin = min(margin, float((running[rest > 0] - draw).abs().min()) if draw > 0 else math.inf)
        got.append(token)
        break
    return got + [-1] * (n - len(got)), len(got) - 1, margin


def check(rt, logits, tokens, runs, u, temperature, draft, more=0, **kw):
    """Every request's result; a row's weight is good to 1e-9, and no decision in these inputs is within 4e-9 of it."""
    starts = torch.tensor([sum(runs[:r]) for r in range(len(runs) + 1)], dtype=torch.int32)
    out = torch.full((len(tokens),), 77, dtype=torch.int32, device="cuda")
    cuda = lambda t: t.cuda() if t is not None else None  # noqa: E731
    got, accepted = rt.verify(logits if logits.is_cuda else logits.cuda(), tokens.cuda(), starts.cuda(), u.cuda(),
                              cuda(temperature), draft if draft is None or draft.is_cuda else draft.cuda(), out=out, **kw)
    got, accepted = got.cpu().tolist(), accepted.cpu().tolist()
    host, hd = logits.cpu(), draft.cpu() if draft is not None else None
    for r, n in enumerate(runs):
        s = int(starts[r])
        if n == 0:
            assert accepted[r] == 0
            continue
        want, count, margin = verified(host[s : s + n], tokens[s : s + n], u[s : s + n].tolist(),
                                       1.0 if temperature is None else float(temperature[r]), hd[s : s + n] if hd is not None else None)
        assert margin > 4e-9, "inputs on a border"
        assert got[s : s + n] == want and accepted[r] == count, (r, got[s : s + n], want)
    assert got[sum(runs):] == [77] * (len(tokens) - sum(runs))


def inputs(rows, requests, vocab, dtype, seed, draft="probabilities", head=True):
    gen = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(rows, vocab, generator=gen)
    if head:
        at = torch.randint(0, vocab, (rows, 12), generator=gen)
        x.scatter_(1, at, 6.0 + 6.0 * torch.rand(rows, 12, generator=gen))
    q = torch.softmax(x + torch.randn(rows, vocab, generator=gen), 1)
    drafted = torch.multinomial(q, 1, generator=gen)[:, 0]
    tokens = torch.cat([drafted.new_zeros(1), drafted[:-1]]).to(torch.int32)
    return (x.to(dtype), tokens, torch.rand(rows, generator=gen), 0.5 + torch.rand(requests, generator=gen),
            q if draft == "probabilities" else q.to(torch.bfloat16) if draft == "bf16" else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", ["probabilities", "bf16", "lookup"])
@pytest.mark.parametrize("runs,vocab", [([1], 1), ([2], 2), ([5, 1, 3], 100), ([8] * 4, 8192), ([4, 0, 6, 1], 8193), ([9, 9], 32003), ([70], 1025)])
def test_verify(rt, dtype, draft, runs, vocab):
    for seed in range(3):
        x, tokens, u, t, q = inputs(sum(runs) + 2, len(runs), vocab, dtype, 100 * seed + vocab, draft, vocab > 50)
        t[0] = 0.0 if seed == 1 else t[0]
        check(rt, x, tokens, runs, u, t, q)


def test_large_vocabulary(rt):
    for vocab in (248320, 1 << 21):
        x, tokens, u, t, q = inputs(6, 2, vocab, torch.float32, vocab, head=False)
        check(rt, x, tokens, [4, 2], u, t, q)


def test_masks_and_ends(rt):
    """Entries of -inf, NaN and +inf, whole rows of them, u at and past its ends, temperatures at theirs, ids that are none."""
    inf, nan = math.inf, math.nan
    x, tokens, u, t, q = inputs(24, 8, 300, torch.float32, 5)
    x[0, ::2], x[1, 5:] = -inf, nan            # masks
    x[3] = -inf                                # a row of nothing at request 1's first row
    x[6, [7, 200]] = inf                       # request 2
    x[9] = 1.5                                 # request 3: all alike
    tokens[7], tokens[13], tokens[16] = 200, -1, 300
    u[11], u[14], u[17], u[20] = 1.0, nan, -3.0, 2.0
    t[3], t[4], t[5], t[6] = inf, 1e-40, nan, -1.0
    q[18, 3] = nan
    for draft in (q, None):
        check(rt, x, tokens, [3] * 8, u, t, draft)
    check(rt, x, tokens, [3] * 8, u, None, q)


def test_the_draft_itself(rt):
    """q equal to p: everything is accepted; q that leaves nothing: drawn from p."""
    x = torch.randn(4, 50, generator=torch.Generator().manual_seed(1))
    tokens = torch.tensor([0, 3, 4, 5], dtype=torch.int32)
    u = torch.tensor([0.3, 0.6, 0.9, 0.5])
    check(rt, x, tokens, [4], u, None, torch.full((4, 50), 1e-9))
    check(rt, x, tokens, [4], u, None, torch.full((4, 50), 2.0))  # (above p everywhere)


def test_layouts_and_graph(rt):
    """Rows of wider and misaligned buffers; a captured call replayed on other inputs, in a workspace of garbage."""
    x, tokens, u, t, q = inputs(12, 3, 9001, torch.bfloat16, 8)
    wide = torch.zeros(12, 9011, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:9004] = x.cuda()
    wide_q = torch.zeros(12, 9020, device="cuda")
    wide_q[:, 1:9002] = q.cuda()
    check(rt, wide[:, 3:9004], tokens, [4, 5, 3], u, t, wide_q[:, 1:9002])
    starts = torch.tensor([0, 4, 9, 12], dtype=torch.int32).cuda()
    ws = torch.full((rt.verify_workspace_bytes(12, 9001, 3),), 0xff, dtype=torch.uint8, device="cuda")
    args = [v.cuda() for v in (x, tokens, starts.cpu(), u, t, q)]
    out, accepted = torch.zeros(12, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    rt.verify(*args, out=out, accepted=accepted, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.verify(*args, out=out, accepted=accepted, workspace=ws)
    for seed in range(4):
        new = inputs(12, 3, 9001, torch.bfloat16, 50 + seed)
        for to, v in zip((args[0], args[1], args[3], args[4], args[5]), new):
            to.copy_(v)
        want = rt.verify(*args)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(accepted, want[1])
        assert bool((ws[:16384] == 0xff).all())


def test_many_draws(rt):
    """Draws over a whole vocabulary, a thousand of them: every token is the one of 64 bits on the host."""
    gen = torch.Generator().manual_seed(4)
    rows, vocab = 256, 100003
    starts = torch.arange(rows + 1, dtype=torch.int32)
    for turn in range(4):
        x = 2.0 * torch.randn(rows, vocab, generator=gen)
        u, t = torch.rand(rows, generator=gen), 0.5 + torch.rand(rows, generator=gen)
        got, _ = rt.verify(x.cuda(), torch.zeros(rows, dtype=torch.int32).cuda(), starts.cuda(), u.cuda(), t.cuda())
        got = got.cpu().long()
        running = ((x.double() - x.amax(1, keepdim=True)) / t.double()[:, None]).exp().cumsum(1)
        draw = u.double()[:, None] * running[:, -1:]
        want = (running > draw).to(torch.uint8).argmax(1)
        # (The order of the sums alone moves a draw by 1e-11 of the weight at most: 100003 additions of 2^-53.)
        for r in (got != want).nonzero()[:, 0].tolist():
            assert abs(float(running[r, min(int(got[r]), int(want[r]))] - draw[r, 0])) < 1e-11 * float(running[r, -1]), (turn, r)
