"""What the Python entry points of the attention layers and of drafted tokens refuse before a launch: shapes, types, devices and
workspaces that do not fit. Outputs stay as they were."""
import pytest
import torch

from splosh_amd._lib import SploshError

pytestmark = pytest.mark.gpu
ROWS, HEADS, KV, DIM, PAGE, VOCAB = 5, 4, 2, 64, 32, 100


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


@pytest.fixture()
def st(rt):
    gen = torch.Generator().manual_seed(1)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    bf = lambda n: torch.randn(ROWS, n, DIM, generator=gen).to(torch.bfloat16).cuda()  # noqa: E731
    cache = rt.Cache.empty(4, PAGE, KV, DIM, "cuda")
    packed = rt.Packed(i32(0, 3, 5), i32(40, 2), torch.tensor([[0, 1], [2, -1]], dtype=torch.int32).cuda())
    return dict(cache=cache, packed=packed, q=bf(HEADS), k=bf(KV), v=bf(KV), f=torch.ones(8).cuda(), w=torch.ones(DIM, dtype=torch.bfloat16).cuda(),
                positions=i32(*range(ROWS)), out=torch.full((ROWS, HEADS, DIM), 3.0, dtype=torch.bfloat16, device="cuda"),
                logits=torch.randn(ROWS, VOCAB, generator=gen).cuda(), tokens=i32(1, 2, 3, 4, 5), u=torch.rand(ROWS).cuda(),
                starts=i32(0, 3, 5))


def refused(call):
    with pytest.raises(SploshError):
        call()


def test_attend(rt, st):
    need = rt.attend_workspace_bytes(st["cache"], st["packed"], ROWS, HEADS)
    run = lambda q=st["q"], **kw: rt.attend(q, st["cache"], st["packed"], out=st["out"], **kw)  # noqa: E731
    for q in (st["q"].float(), st["q"].cpu(), st["q"][0], st["q"][:, :3], st["q"][..., :32], st["q"].transpose(1, 2).contiguous().transpose(1, 2),
              st["q"][:, :0], st["q"][:0]):
        refused(lambda: run(q))
    for kw in (dict(rows=ROWS + 1), dict(rows=0), dict(shared=5), dict(shared=-32), dict(shared=96), dict(scale=0.0), dict(scale=float("nan")),
               dict(workspace=torch.zeros(need - 1, dtype=torch.uint8, device="cuda")), dict(workspace=torch.zeros(need, dtype=torch.uint8)),
               dict(workspace=torch.zeros(2 * need, dtype=torch.uint8, device="cuda")[::2])):
        refused(lambda: run(**kw))
    for out in (st["out"].float(), st["out"][:4], st["out"].cpu(), torch.zeros(ROWS, HEADS, 2 * DIM, dtype=torch.bfloat16, device="cuda")[..., :DIM]):
        refused(lambda: rt.attend(st["q"], st["cache"], st["packed"], out=out))
    assert bool((st["out"] == 3).all())


def test_workspace_of_long_prompts(rt, st):
    """Beside sixteen bytes a (row, query head) the scratch is a matter of the device, not of the prompt's length."""
    one = rt.Packed(st["packed"].starts[:2].contiguous(), st["packed"].lengths[:1].contiguous(), st["packed"].table[:1].contiguous())
    need = {rows: rt.attend_workspace_bytes(st["cache"], one, rows, HEADS) for rows in (2048, 1 << 17)}
    assert need[1 << 17] - need[2048] == 16 * HEADS * ((1 << 17) - 2048)


def test_heads_and_cache(rt, st):
    write = lambda k=st["k"], v=st["v"], q=st["q"], **kw: rt.cache_write(st["cache"], st["packed"], k, v, q, out=st["out"], **kw)  # noqa: E731
    for kw in (dict(k=st["q"]), dict(v=st["v"].float()), dict(q=st["q"].float()), dict(k=st["k"].cpu()), dict(v=st["v"][:4]), dict(q=st["q"][..., :32]),
               dict(k_weight=st["w"][:10]), dict(k_weight=st["w"].float()), dict(q_weight=st["w"].cpu()), dict(frequencies=st["f"].double()),
               dict(frequencies=torch.ones(33).cuda()), dict(frequencies=st["f"].cpu()), dict(rows=6), dict(rows=-1)):
        refused(lambda: write(**kw))
    rotate = lambda xs=(st["q"], st["k"]), positions=st["positions"], f=st["f"], **kw: rt.rotate_heads(xs, positions, f, **kw)  # noqa: E731
    for kw in (dict(xs=()), dict(xs=[st["q"]] * 9), dict(xs=(st["q"], st["k"].float())), dict(positions=st["positions"].long()),
               dict(positions=st["positions"][:4]), dict(positions=None), dict(weights=[st["w"]]), dict(outs=[st["out"]]), dict(rows=6),
               dict(f=torch.ones(33).cuda()), dict(xs=(st["q"][..., :48],))):
        refused(lambda: rotate(**kw))
    for kw in (dict(), dict(rows=0), dict(k=st["out"]), dict(v=st["k"].float()), dict(rows=6, k=st["k"])):
        refused(lambda: rt.cache_read(st["cache"], st["packed"], **kw))
    assert bool((st["out"] == 3).all()) and not st["cache"].data.any()


def test_handles(rt, st):
    p, c = st["packed"], st["cache"]
    for make in (lambda: rt.Packed(p.starts.long(), p.lengths, p.table), lambda: rt.Packed(p.starts[:2], p.lengths, p.table),
                 lambda: rt.Packed(p.starts, p.lengths.cpu(), p.table), lambda: rt.Packed(p.starts, p.lengths, p.table.t()),
                 lambda: rt.Packed(p.starts, p.lengths, p.table[0]), lambda: rt.Packed(p.starts, p.lengths, p.table.float()),
                 lambda: rt.Cache(c.data, 48, KV, DIM), lambda: rt.Cache(c.data, PAGE, KV, 96), lambda: rt.Cache(c.data, PAGE, 0, DIM),
                 lambda: rt.Cache(c.data[:, :-16], PAGE, KV, DIM), lambda: rt.Cache(c.data.cpu(), PAGE, KV, DIM),
                 lambda: rt.Cache(c.data.int(), PAGE, KV, DIM), lambda: rt.Cache(c.data[0], PAGE, KV, DIM)):
        refused(make)


def test_verify(rt, st):
    out, accepted = (torch.full((n,), 7, dtype=torch.int32, device="cuda") for n in (ROWS, 2))
    base = dict(logits=st["logits"], tokens=st["tokens"], starts=st["starts"], uniforms=st["u"])
    need = rt.verify_workspace_bytes(ROWS, VOCAB, 2)
    for kw in (dict(logits=st["logits"].half()), dict(logits=st["logits"].t()), dict(logits=st["logits"].cpu()), dict(tokens=st["tokens"].long()),
               dict(tokens=st["tokens"][:4]), dict(starts=st["starts"][:1]), dict(starts=st["starts"].cpu()), dict(uniforms=st["u"].double()),
               dict(temperature=st["u"][:1]), dict(draft=st["logits"][:4]), dict(draft=st["logits"][:, :99]), dict(draft=st["logits"].half()),
               dict(out=out[:4]), dict(accepted=accepted.long()), dict(workspace=torch.zeros(need - 1, dtype=torch.uint8, device="cuda")),
               dict(workspace=torch.zeros(need, dtype=torch.uint8))):
        refused(lambda: rt.verify(**{**base, "out": out, "accepted": accepted, **kw}))
    assert bool((out == 7).all()) and bool((accepted == 7).all())
