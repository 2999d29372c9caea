"""The attention operators and the verification of drafted tokens together with the projections around them, as a serving
loop runs them: tokens -> embedding -> q, k, v -> norm, rotation and cache -> attention -> out projection onto the
residual (two layers) -> lm_head -> verification, whose tokens the next step embeds. Eager and as one captured graph, every stage
against its definition on what the stage before it gave."""
import pytest
import torch

from qcheck import Q4Case
from step_check import attended, check_bf16, kept, rotated
from test_gpu_verify import verified

pytestmark = pytest.mark.gpu
HIDDEN, Q, KV, DIM, VOCAB, PAGE, LAYERS, ROTARY = 512, 6, 2, 128, 2048, 32, 2, 64
PROMPTS, DRAFTED, EPS = (40, 9, 33), 3, 1e-6
REQUESTS = len(PROMPTS)
PAGES = 24


class Model:
    def __init__(self, rt):
        self.rt = rt
        self.table, self.head = Q4Case(VOCAB, HIDDEN, seed=1), Q4Case(VOCAB, HIDDEN, seed=2)
        gen = torch.Generator().manual_seed(3)
        self.layers, self.norms = [], []
        for i in range(LAYERS):
            self.layers.append([Q4Case(n, k, seed=10 * i + j) for j, (n, k) in enumerate(
                ((Q * DIM, HIDDEN), (KV * DIM, HIDDEN), (KV * DIM, HIDDEN), (HIDDEN, Q * DIM)), 4)])
            self.norms.append([(1 + 0.2 * torch.randn(DIM, generator=gen)).to(torch.bfloat16) for _ in "qk"])
        self.frequencies = (1.0e6 ** (-torch.arange(ROTARY // 2) / (ROTARY // 2))).float()
        self.on_gpu = self.frequencies.cuda(), [[w.cuda() for w in pair] for pair in self.norms]
        order = torch.randperm(PAGES, generator=gen).to(torch.int32)
        self.pages = order.view(REQUESTS, -1)
        self.reset()

    def reset(self):
        self.caches = [self.rt.Cache.empty(PAGES, PAGE, KV, DIM, "cuda") for _ in range(LAYERS)]

    def packed(self, runs, lengths):
        starts = torch.tensor([sum(runs[:r]) for r in range(REQUESTS + 1)], dtype=torch.int32)
        return self.rt.Packed(starts.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), self.pages.cuda())

    def workspace(self, packed, rows):
        """One zeroed scratch for every call of a step."""
        rt = self.rt
        need = [rt.workspace_bytes(rows, n, k) for n, k in (((Q + 2 * KV) * DIM, HIDDEN), (HIDDEN, Q * DIM), (VOCAB, HIDDEN))]
        need += [rt.attend_workspace_bytes(self.caches[0], packed, rows, Q), rt.verify_workspace_bytes(rows, VOCAB, REQUESTS)]
        return torch.zeros(max(need), dtype=torch.uint8, device="cuda")

    def step(self, tokens, packed, ws, keep=lambda *_: None):
        """One step's logits; `keep`: called with each layer's tensors."""
        rt, (frequencies, norms) = self.rt, self.on_gpu
        rows = tokens.numel()
        hidden = rt.embed(self.table.w_tiled, tokens)
        for i, (wq, wk, wv, wo) in enumerate(self.layers):
            x, _ = rt.prepare_operand(hidden)
            q, k, v = (t.view(rows, -1, DIM) for t in rt.gemm_group([wq.w_tiled, wk.w_tiled, wv.w_tiled], x, out_dtype=torch.float32,
                                                                   workspace=ws))
            turned = rt.cache_write(self.caches[i], packed, k, v, q, frequencies, norms[i][1], norms[i][0], EPS)
            mixed = rt.attend(turned, self.caches[i], packed, workspace=ws)
            keep(i, q, k, v, turned, mixed)
            rt.gemm(wo.w_tiled, mixed.view(rows, -1), out=hidden, residual=hidden, workspace=ws)
        y, _ = rt.prepare_operand(hidden)
        return rt.gemm(self.head.w_tiled, y, out_dtype=torch.float32, workspace=ws)

    def held(self, i, r, n):
        """Keys and values of request r's first n tokens from the bytes of layer i's cache, in 64 bits."""
        data = self.caches[i].data.cpu().view(PAGES, KV, PAGE // 32, 64 * DIM + 256)[self.pages[r].long()]
        codes = data[..., : 64 * DIM].reshape(-1, KV, PAGE // 32, 2, 32, DIM).double() - 128
        scales = data[..., 64 * DIM :].contiguous().view(torch.float32).view(-1, KV, PAGE // 32, 2, 32, 1).double()
        both = (codes * scales).permute(3, 0, 2, 4, 1, 5).reshape(2, -1, KV, DIM)
        return both[0, :n], both[1, :n]

    def check_layer(self, i, runs, lengths, q, k, v, turned, mixed):
        q, k, v, turned, mixed = (t.cpu() for t in (q, k, v, turned, mixed))
        positions = torch.cat([torch.arange(n - m, n) for m, n in zip(runs, lengths)])
        want, off = rotated(q, self.norms[i][0], self.frequencies, positions, EPS)
        check_bf16(turned, want, off, f"queries of layer {i}")
        want_k, off_k = rotated(k, self.norms[i][1], self.frequencies, positions, EPS)
        begin = 0
        for r, (m, n) in enumerate(zip(runs, lengths)):
            rows = slice(begin, begin + m)
            keys, values = self.held(i, r, n)
            for got, x, more in ((keys[n - m :], want_k[rows], off_k[rows]), (values[n - m :], v[rows].double(), torch.zeros(1))):
                _, scale = kept(x)  # half a step, and what fp32 leaves of the vector and of its largest
                assert bool(((got - x).abs() <= scale * (0.5 + 2.0 ** -14) + more + more.amax(-1, keepdim=True)).all())
            out, off = attended(turned[rows], keys, values, torch.arange(n - m, n), DIM ** -0.5)
            check_bf16(mixed[rows], out, off, f"request {r} of layer {i}")
            begin += m


@pytest.fixture(scope="module")
def model():
    from splosh_amd import runtime as rt
    return Model(rt)


def check_verified(model, logits, tokens, runs, u, temperature, out, accepted):
    begin = 0
    for r, m in enumerate(runs):
        rows = slice(begin, begin + m)
        want, count, margin = verified(logits[rows].cpu(), tokens[rows], u[rows].tolist(), float(temperature[r]), None)
        assert margin > 4e-9
        assert out[rows].tolist() == want and int(accepted[r]) == count
        begin += m


def test_a_prompt_and_verify_steps(model):
    """Prompts of three lengths, then steps of one token and three drafted ones each; drafts are what the step before it would
    have drawn (request 0 is greedy, so its first one is accepted when the step is run again)."""
    model.reset()
    gen = torch.Generator().manual_seed(9)
    ids = torch.randint(0, VOCAB, (sum(PROMPTS),), generator=gen, dtype=torch.int32)
    lengths, runs = list(PROMPTS), list(PROMPTS)
    tokens, temperature = ids, torch.tensor([0.0, 0.8, 1.3])
    for step in range(5):
        rows = sum(runs)
        packed, u = model.packed(runs, lengths), torch.rand(rows, generator=gen)
        ws = model.workspace(packed, rows)
        logits = model.step(tokens.cuda(), packed, ws, lambda i, *t: model.check_layer(i, runs, lengths, *t))
        out, accepted = model.rt.verify(logits, tokens.cuda(), packed.starts, u.cuda(), temperature.cuda(), workspace=ws)
        out, accepted = out.cpu(), accepted.cpu()
        assert not ws[: model.rt.WORKSPACE_COUNTER_BYTES].any()
        if step == 0:  # (a prompt: its last row draws the next token)
            picked = [int(logits[sum(runs[: r + 1]) - 1].argmax()) for r in range(REQUESTS)]
            taken = [0] * REQUESTS
        else:
            check_verified(model, logits, tokens, runs, u, temperature, out, accepted)
            begins = [sum(runs[:r]) for r in range(REQUESTS)]
            taken = accepted.tolist()
            picked = [int(out[b + n]) for b, n in zip(begins, taken)]
            if step in (2, 4):
                assert taken[0] >= 1
        if step in (1, 3):  # the same step again, with the greedy request's token as its first draft
            tokens = tokens.clone()
            tokens[taken[0] + 1] = picked[0]
            continue
        lengths = [n + (0 if step == 0 else t + 1 - m) + 1 + DRAFTED for n, t, m in zip(lengths, taken, runs)]
        runs = [1 + DRAFTED] * REQUESTS
        drafts = torch.randint(0, VOCAB, (REQUESTS, DRAFTED), generator=gen, dtype=torch.int32)
        tokens = torch.cat([torch.cat([torch.tensor([p], dtype=torch.int32), d]) for p, d in zip(picked, drafts)])


def test_captured_step(model):
    """A verify step as one graph: tokens, lengths and uniforms change between the replays, with eager work between them; every
    replay gives the eager step's logits, tokens and caches bit for bit."""
    model.reset()
    rt, rows = model.rt, REQUESTS * (1 + DRAFTED)
    runs = [1 + DRAFTED] * REQUESTS
    gen = torch.Generator().manual_seed(11)
    for cache in model.caches:  # a past of random tokens
        k, v = (torch.randn(PAGES * PAGE, KV, DIM, generator=gen).to(torch.bfloat16).cuda() for _ in "kv")
        ends = torch.tensor([0, PAGES * PAGE], dtype=torch.int32).cuda()
        rt.cache_write(cache, rt.Packed(ends, ends[1:].clone(), torch.arange(PAGES, dtype=torch.int32).cuda()[None]), k, v)
    packed = model.packed(runs, [100, 4, 77])
    ws = model.workspace(packed, rows)
    tokens, u = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    temperature = torch.tensor([0.0, 0.7, 1.0]).cuda()

    def whole():
        logits = model.step(tokens, packed, ws)
        return logits, *rt.verify(logits, tokens, packed.starts, u, temperature, workspace=ws)

    whole()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = whole()
    for lengths in ([100, 4, 77], [104, 5, 256], [64, 33, 80], [100, 4, 77]):
        packed.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        tokens.copy_(torch.randint(0, VOCAB, (rows,), generator=gen, dtype=torch.int32))
        u.copy_(torch.rand(rows, generator=gen))
        before = [c.data.clone() for c in model.caches]
        want = whole()
        after = [c.data.clone() for c in model.caches]
        torch.cuda.synchronize()
        for cache, data in zip(model.caches, before):
            cache.data.copy_(data)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.int32), b.view(torch.int32)), lengths
        for cache, data in zip(model.caches, after):
            assert torch.equal(cache.data, data), lengths
        check_verified(model, got[0], tokens.cpu(), runs, u.cpu(), temperature.cpu(), got[1].cpu(), got[2].cpu())
    assert not ws[: rt.WORKSPACE_COUNTER_BYTES].any()


def test_two_graphs_one_workspace(model):
    """Two captured steps of different shapes that share a workspace, replayed in turn."""
    model.reset()
    rt = model.rt
    gen = torch.Generator().manual_seed(12)
    cache = model.caches[0]
    steps = []
    for runs, lengths in (([1, 1, 1], [200, 31, 250]), ([70, 3, 1], [70, 250, 128])):
        packed, rows = model.packed(runs, lengths), sum(runs)
        k, v, q = (torch.randn(rows, n, DIM, generator=gen).cuda() for n in (KV, KV, Q))
        steps.append((packed, rows, k, v, q))
    ws = torch.zeros(max(rt.attend_workspace_bytes(cache, s[0], s[1], Q) for s in steps), dtype=torch.uint8, device="cuda")

    def run(packed, rows, k, v, q):
        return rt.attend(rt.cache_write(cache, packed, k, v, q), cache, packed, workspace=ws)

    graphs = []
    for s in steps:
        run(*s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(*s)
        graphs.append((g, out))
    for turn in range(3):
        for s, (g, out) in zip(steps, graphs):
            s[4].copy_(torch.randn(s[4].shape, generator=gen))
            want = run(*s)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), turn


def test_side_streams(model):
    """Every call on another stream than the current one, its tensors made there."""
    model.reset()
    rt = model.rt
    gen = torch.Generator().manual_seed(13)
    packed = model.packed([2, 1, 4], [64, 40, 4])
    k, v, q = (torch.randn(7, n, DIM, generator=gen).to(torch.bfloat16).cuda() for n in (KV, KV, Q))
    logits, u = torch.randn(7, VOCAB, generator=gen).cuda(), torch.rand(7, generator=gen).cuda()
    tokens = torch.randint(0, VOCAB, (7,), generator=gen, dtype=torch.int32).cuda()
    f, norms = model.on_gpu[0], model.on_gpu[1][0]
    positions = torch.arange(7, dtype=torch.int32).cuda()

    def run(stream):
        cache = rt.Cache.empty(PAGES, PAGE, KV, DIM, "cuda")
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        turned = rt.cache_write(cache, packed, k, v, q, f, norms[1], norms[0], EPS, stream=stream)
        back = rt.cache_read(cache, packed, 7, stream=stream)
        got = [turned, *back, rt.attend(turned, cache, packed, stream=stream), *rt.rotate_heads([q, k], positions, f, norms, stream=stream),
               *rt.verify(logits, tokens, packed.starts, u, stream=stream)]
        if stream is not None:
            torch.cuda.current_stream().wait_stream(stream)
        return got

    want = run(None)
    torch.cuda.synchronize()
    for a, b in zip(run(torch.cuda.Stream()), want):
        assert torch.equal(a, b)
