"""The per-request operators together with the projections of a packed step, as a serving loop runs
them: tokens -> embedding -> gate and up with adapters -> silu(gate) * up -> down with adapters onto the
residual -> lm_head with adapters -> the next tokens, which the next step embeds. Eager and as one
captured graph, every stage against its definition on what the stage before it gave."""
import pytest
import torch

from adapter_check import check
from qcheck import Q4Case
from sample_check import check_row

pytestmark = pytest.mark.gpu
HIDDEN, INTER, VOCAB, RANK, SLOTS, ROWS = 512, 1024, 4096, 16, 4, 24


class Model:
    def __init__(self, rt):
        self.rt = rt
        self.table, self.gate, self.up = (Q4Case(n, HIDDEN, seed=s) for n, s in ((VOCAB, 1), (INTER, 2), (INTER, 3)))
        self.down, self.head = Q4Case(HIDDEN, INTER, seed=4), Q4Case(VOCAB, HIDDEN, seed=5)
        gen = torch.Generator().manual_seed(6)
        self.host, self.adapters = {}, {}
        for name, n, k in (("gate", INTER, HIDDEN), ("up", INTER, HIDDEN), ("down", HIDDEN, INTER), ("head", VOCAB, HIDDEN)):
            a = (torch.randn(SLOTS, RANK, k, generator=gen) / k ** 0.5).to(torch.bfloat16)
            b = (0.1 * torch.randn(SLOTS, n, RANK, generator=gen)).to(torch.bfloat16)
            scales = 0.5 + torch.rand(SLOTS, generator=gen)
            ranks = torch.tensor([RANK, 5, 0, RANK], dtype=torch.int32)
            self.host[name] = (a, b, scales, ranks)
            self.adapters[name] = rt.Adapters(a.cuda(), b.cuda(), scales.cuda(), ranks.cuda())
        # One zeroed scratch for every call of the step.
        need = [rt.workspace_bytes(ROWS, n, k) for n, k in ((2 * INTER, HIDDEN), (HIDDEN, INTER), (VOCAB, HIDDEN))]
        need += [rt.adapters_workspace_bytes([self.adapters["gate"], self.adapters["up"]], ROWS),
                 rt.adapters_workspace_bytes(self.adapters["down"], ROWS),
                 rt.adapters_workspace_bytes(self.adapters["head"], ROWS), rt.sample_workspace_bytes(ROWS, VOCAB)]
        self.ws = torch.zeros(max(need), dtype=torch.uint8, device="cuda")

    def step(self, tokens, slots, u, params, keep):
        """One step; `keep`: called with each stage's name and tensors."""
        rt, ws = self.rt, self.ws
        hidden = rt.embed(self.table.w_tiled, tokens)
        x, _ = rt.prepare_operand(hidden)
        both = rt.gemm_group([self.gate.w_tiled, self.up.w_tiled], x, out_dtype=torch.float32, workspace=ws)
        keep("gate_up", x, both)
        rt.add_adapters_group(both, x, [self.adapters["gate"], self.adapters["up"]], slots, workspace=ws)
        keep("gate_up_adapted", x, both)
        act, _ = rt.silu_mul_operand(*both)
        rt.gemm(self.down.w_tiled, act, out=hidden, residual=hidden, workspace=ws)
        keep("down", act, [hidden])
        rt.add_adapters(hidden, act, self.adapters["down"], slots, workspace=ws)
        keep("down_adapted", act, [hidden])
        y, _ = rt.prepare_operand(hidden)
        logits = rt.gemm(self.head.w_tiled, y, out_dtype=torch.float32, workspace=ws)
        keep("head", y, [logits])
        rt.add_adapters(logits, y, self.adapters["head"], slots, workspace=ws)
        keep("head_adapted", y, [logits])
        return rt.sample(logits, u, **params, workspace=ws) + (logits,)


@pytest.fixture(scope="module")
def model():
    from splosh_amd import runtime as rt
    return Model(rt)


def inputs(seed):
    gen = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, VOCAB, (ROWS,), generator=gen, dtype=torch.int32)
    slots = (torch.arange(ROWS) // 4 - 1).to(torch.int32)  # requests of four rows; the first and last without
    u = torch.rand(ROWS, generator=gen)
    params = {"temperature": torch.where(torch.arange(ROWS) % 3 == 0, torch.tensor(0.0), torch.tensor(0.9)),
              "top_k": torch.where(torch.arange(ROWS) % 2 == 0, 0, 40).to(torch.int32),
              "top_p": torch.where(torch.arange(ROWS) % 5 == 0, torch.tensor(1.0), torch.tensor(0.9))}
    return tokens, slots, u, params


def check_sampled(logits, tokens, logprobs, u, params):
    for r in range(ROWS):
        check_row(logits[r].cpu().numpy(), tokens[r], float(logprobs[r]), float(u[r]),
                  **{n: v[r].item() for n, v in params.items()}, label=f"row {r}")


def test_steps(model):
    tokens, slots, u, params = inputs(7)
    tokens = tokens.cuda()
    for _ in range(3):
        seen = {}
        got = model.step(tokens, slots.cuda(), u.cuda(), {n: v.cuda() for n, v in params.items()},
                         lambda name, x, outs: seen.update({name: (x.cpu(), [o.cpu() for o in outs])}))
        for stage, names in (("gate_up", ("gate", "up")), ("down", ("down",)), ("head", ("head",))):
            x, before = seen[stage]
            for name, b, after in zip(names, before, seen[stage + "_adapted"][1]):
                check(after, b, x, model.host[name], slots, name)
        check_sampled(got[2], got[0].cpu(), got[1].cpu(), u, params)
        assert not model.ws[: model.rt.WORKSPACE_COUNTER_BYTES].any()
        tokens = got[0]


def test_captured_step(model):
    """The step as one graph that feeds itself: each replay embeds the tokens the last one drew. Every
    replay equals the eager step from the same tokens."""
    tokens, slots, u, params = inputs(8)
    tokens, slots, ud = tokens.cuda(), slots.cuda(), u.cuda()
    dev = {n: v.cuda() for n, v in params.items()}
    nothing = lambda *_: None  # noqa: E731
    model.step(tokens, slots, ud, dev, nothing)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, logprobs, logits = model.step(tokens, slots, ud, dev, nothing)
        tokens.copy_(out)
    for k in range(4):
        start = tokens.clone()
        want = model.step(start, slots, ud, dev, nothing)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits.view(torch.int32), want[2].view(torch.int32)), f"replay {k}"
        assert torch.equal(out, want[0]) and torch.equal(logprobs, want[1]), f"replay {k}"
        assert torch.equal(tokens, out)
        check_sampled(logits, out.cpu(), logprobs.cpu(), u, params)
