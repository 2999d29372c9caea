"""splosh_adapters_add / _group against their formula in 64 bits: every rank, length and layout, rows
without an adapter, and what must stay as it was."""
import pytest
import torch

from adapter_check import check

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def host_case(rows, inner, outputs, rank, count, dtype, seed, ranks=None):
    """Inputs on the host: x, (a, b, scales, ranks), out before."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen)

    x = normal(rows, inner).to(torch.bfloat16)
    a = (normal(count, rank, inner) / inner ** 0.5).to(torch.bfloat16)
    b = (normal(count, outputs, rank) * 0.1).to(torch.bfloat16)
    scales = 0.5 + torch.rand(count, generator=gen)
    out = normal(rows, outputs).to(dtype)
    return x, (a, b, scales, None if ranks is None else torch.tensor(ranks, dtype=torch.int32)), out


def slots_of(rows, count, seed, spread="rows"):
    gen = torch.Generator().manual_seed(seed + 1000)
    if spread == "one":
        return torch.zeros(rows, dtype=torch.int32)
    if spread == "runs":
        return (torch.arange(rows) * count // max(rows, 1)).to(torch.int32)
    return torch.randint(-1, count + 1, (rows,), generator=gen).to(torch.int32)  # both kinds of "none" too


def on_gpu(rt, adapters):
    a, b, scales, ranks = adapters
    return rt.Adapters(a.cuda(), b.cuda(), None if scales is None else scales.cuda(), None if ranks is None else ranks.cuda())


def run(rt, case, slots, label=""):
    x, adapters, out = case
    got = out.cuda()
    assert rt.add_adapters(got, x.cuda(), on_gpu(rt, adapters), slots.cuda()) is got
    check(got, out, x, adapters, slots, label)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 7, 16, 17, 33, 63, 64, 65, 128, 200, 333])
def test_row_counts(rt, rows, dtype):
    for spread in ("rows", "one", "runs"):
        run(rt, host_case(rows, 320, 200, 16, 5, dtype, rows), slots_of(rows, 5, rows, spread), f"{rows} {spread}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [1, 2, 3, 5, 8, 12, 16, 17, 24, 31, 32, 33, 48, 64, 65, 100, 128, 200, 256])
def test_ranks(rt, rank, dtype):
    for rows in (3, 70):
        run(rt, host_case(rows, 264, 136, rank, 3, dtype, rank), slots_of(rows, 3, rank), f"rank {rank} rows {rows}")


@pytest.mark.parametrize("inner", [1, 2, 7, 8, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 500, 512, 1001, 1536, 4352])
def test_inner_sizes(rt, inner):
    for rows, dtype in ((1, torch.float32), (20, torch.bfloat16), (80, torch.float32)):
        run(rt, host_case(rows, inner, 72, 16, 3, dtype, inner), slots_of(rows, 3, inner), f"inner {inner} rows {rows}")


@pytest.mark.parametrize("outputs", [1, 2, 7, 15, 16, 17, 63, 64, 65, 100, 255, 256, 257, 513, 1000, 2049])
def test_output_sizes(rt, outputs):
    for rows, dtype in ((1, torch.bfloat16), (20, torch.float32), (80, torch.bfloat16)):
        run(rt, host_case(rows, 96, outputs, 16, 3, dtype, outputs), slots_of(rows, 3, outputs),
            f"outputs {outputs} rows {rows}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 8, 64, 160])
def test_long_inner(rt, rows, dtype):
    """The lengths of real projections, split over many workgroups."""
    run(rt, host_case(rows, 17408, 640, 16, 4, dtype, rows), slots_of(rows, 4, rows), f"rows {rows}")
    run(rt, host_case(rows, 5120, 5120, 64, 4, dtype, rows), slots_of(rows, 4, rows), f"wide, rows {rows}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_ranks_of_slots(rt, dtype):
    """Each slot its own rank: 0 and below leave the row, above max_rank counts as it, and what lies
    past a rank (NaN here) is never used."""
    ranks = [0, 1, 5, 16, 17, 40, 41, 1000, -3]
    x, (a, b, scales, r), out = host_case(90, 200, 150, 41, len(ranks), dtype, 3, ranks)
    for s, n in enumerate(ranks):
        a[s, max(n, 0):] = float("nan")
        b[s, :, max(n, 0):] = float("nan")
    run(rt, (x, (a, b, scales, r), out), slots_of(90, len(ranks), 4))


@pytest.mark.parametrize("rows", [1, 24, 100])
def test_defaults(rt, rows):
    """No scales (1) and no ranks (max_rank)."""
    x, (a, b, _, _), out = host_case(rows, 128, 80, 8, 3, torch.float32, 9)
    run(rt, (x, (a, b, None, None), out), slots_of(rows, 3, 9))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 20, 70])
@pytest.mark.parametrize("pad", [1, 2, 8])
def test_strides(rt, rows, pad, dtype):
    """Operands that are parts of wider buffers, at odd places and odd strides; what surrounds them
    (NaN) is neither used nor written."""
    inner, outputs, rank, count = 136, 104, 16, 3
    x, adapters, out = host_case(rows, inner, outputs, rank, count, dtype, pad)
    a, b, scales, _ = adapters

    def part(t):
        shape = [n + pad for n in t.shape]
        wide = torch.full(shape, float("nan"), dtype=t.dtype, device="cuda")
        view = wide[tuple(slice(pad, None) for _ in shape)]
        view.copy_(t)
        return wide, view

    slots = slots_of(rows, count, pad)
    wide_out, got = part(out)
    before = wide_out.clone()
    rt.add_adapters(got, part(x)[1], rt.Adapters(part(a)[1], part(b)[1], part(scales)[1]), part(slots.float())[1].int())
    check(got, out, x, adapters, slots)
    before[pad:, pad:] = got
    same = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(wide_out.view(same), before.view(same)), "written outside the output"


def test_slots_shared_by_stride(rt):
    """A slot stride of 0: every slot the same matrices, with its own scale."""
    x, (a, b, scales, _), out = host_case(40, 64, 48, 8, 4, torch.float32, 11)
    a, b = a[:1].expand(4, -1, -1), b[:1].expand(4, -1, -1)
    slots = slots_of(40, 4, 11)
    got = out.cuda()
    rt.add_adapters(got, x.cuda(), rt.Adapters(a[:1].cuda().expand(4, -1, -1), b[:1].cuda().expand(4, -1, -1), scales.cuda()),
                    slots.cuda())
    check(got, out, x, (a, b, scales, None), slots)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 8, 64, 90, 260])
def test_group(rt, rows, dtype):
    """Several projections of one activation, of different widths, ranks and slot counts: the same
    result as one call each, to the bit where the split is the same, and each against the formula."""
    shapes = [(256, 16, 6), (64, 16, 6), (65, 40, 4), (1, 3, 9)]
    cases = [host_case(rows, 640, n, r, c, dtype, i) for i, (n, r, c) in enumerate(shapes)]
    x = cases[0][0]
    slots = slots_of(rows, 6, rows)
    outs = [c[2].cuda() for c in cases]
    back = rt.add_adapters_group(outs, x.cuda(), [on_gpu(rt, c[1]) for c in cases], slots.cuda())
    assert all(p is q for p, q in zip(back, outs))
    for i, (c, got) in enumerate(zip(cases, outs)):
        check(got, c[2], x, c[1], slots, f"projection {i}")


def test_group_of_eight(rt):
    cases = [host_case(30, 200, 40 + i, 8, 3, torch.float32, i) for i in range(8)]
    slots = slots_of(30, 3, 1)
    outs = [c[2].cuda() for c in cases]
    rt.add_adapters_group(outs, cases[0][0].cuda(), [on_gpu(rt, c[1]) for c in cases], slots.cuda())
    for c, got in zip(cases, outs):
        check(got, c[2], cases[0][0], c[1], slots)


@pytest.mark.parametrize("rows", [64, 150])
def test_every_row_its_own_adapter(rt, rows):
    case = host_case(rows, 256, 96, 8, rows, torch.float32, 21)
    run(rt, case, torch.randperm(rows, generator=torch.Generator().manual_seed(5)).to(torch.int32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [5, 64, 100])
def test_nonfinite_rows_stay_their_own(rt, rows, dtype):
    """An infinite or NaN activation makes its own row's outputs non-finite (infinities where every
    product with it is one) and no other's."""
    x, adapters, out = host_case(rows, 96, 80, 16, 3, dtype, 31)
    slots = slots_of(rows, 3, 31, "one")
    x[1, 5], x[3, 90] = float("inf"), float("nan")
    adapters[0][0, :, 5] = adapters[0][0, :, 5].abs() + 0.5
    adapters[1][0] = adapters[1][0].abs() + 0.25
    got = out.cuda()
    rt.add_adapters(got, x.cuda(), on_gpu(rt, adapters), slots.cuda())
    got = got.cpu()
    assert torch.isinf(got[1]).all() and (got[1] > 0).all() and torch.isnan(got[3]).all()
    rest = [m for m in range(rows) if m not in (1, 3)]
    check(got[rest].cuda(), out[rest], x[rest], adapters, slots[rest])


def test_many_rows(rt):
    """More rows than any launch dimension of 65535 takes."""
    rows = 66000
    x, adapters, out = host_case(rows, 16, 4, 4, 3, torch.float32, 41)
    slots = slots_of(rows, 3, 41)
    got = out.cuda()
    rt.add_adapters(got, x.cuda(), on_gpu(rt, adapters), slots.cuda())
    pick = list(range(0, 300)) + list(range(65400, 66000))
    check(got[pick], out[pick], x[pick], adapters, slots[pick])


def test_far_offsets(rt):
    """Rows and slots whose elements lie past 2^32 bytes."""
    count, rank, inner, outputs = 3, 8, 64, 64
    a = torch.zeros(count, 1 << 28, dtype=torch.uint8, device="cuda")  # only to be the distance
    far = torch.zeros(3 * (1 << 30), dtype=torch.bfloat16, device="cuda")
    del a
    x, adapters, out = host_case(40, inner, outputs, rank, count, torch.bfloat16, 51)
    a = far.as_strided((count, rank, inner), (1 << 30, inner, 1))
    b = far.as_strided((count, outputs, rank), (1 << 30, rank, 1), 4096)
    got = far.as_strided((40, outputs), (75_000_000, 1), 8192)
    a.copy_(adapters[0].cuda())
    b.copy_(adapters[1].cuda())
    got.copy_(out.cuda())
    slots = slots_of(40, count, 51)
    rt.add_adapters(got, x.cuda(), rt.Adapters(a, b, adapters[2].cuda()), slots.cuda())
    check(got, out, x, adapters, slots)


def test_streams_and_shared_workspace(rt):
    """Two streams with a workspace each, and one workspace that other entry points use before and
    after: the counters at its start are left alone."""
    cases = [host_case(48, 512, 320, 16, 4, torch.float32, s) for s in (61, 62)]
    slots = slots_of(48, 4, 61)
    devs = [(c[0].cuda(), on_gpu(rt, c[1]), c[2].cuda(), slots.cuda()) for c in cases]
    streams = [torch.cuda.Stream() for _ in devs]
    torch.cuda.synchronize()
    for s, (x, w, out, sl) in zip(streams, devs):
        rt.add_adapters(out, x, w, sl, stream=s)
    torch.cuda.synchronize()
    for c, d in zip(cases, devs):
        check(d[2], c[2], c[0], c[1], slots)
    ws = torch.zeros(max(rt.adapters_workspace_bytes(devs[0][1], 48), rt.workspace_bytes(48, 320, 512)), dtype=torch.uint8,
                     device="cuda")
    got = cases[0][2].cuda()
    rt.add_adapters(got, devs[0][0], devs[0][1], devs[0][3], workspace=ws)
    check(got, cases[0][2], cases[0][0], cases[0][1], slots)
    assert not ws[: rt.WORKSPACE_COUNTER_BYTES].any()


def test_graph_replays(rt):
    """Captured together and replayed with other adapters, slots and rows written into the same tensors:
    every replay is the eager result of the same inputs."""
    x, adapters, out = host_case(24, 640, 200, 16, 4, torch.bfloat16, 71)
    w, xd, buf = on_gpu(rt, adapters), x.cuda(), out.cuda()
    slots = slots_of(24, 4, 71).cuda()
    ws = torch.zeros(rt.adapters_workspace_bytes(w, 24), dtype=torch.uint8, device="cuda")
    rt.add_adapters(buf.clone(), xd, w, slots, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.add_adapters(buf, xd, w, slots, workspace=ws)
    for seed in range(72, 76):
        nx, nw, nout = host_case(24, 640, 200, 16, 4, torch.bfloat16, seed)
        xd.copy_(nx), w.a.copy_(nw[0]), w.b.copy_(nw[1]), w.scales.copy_(nw[2]), buf.copy_(nout)
        slots.copy_(slots_of(24, 4, seed))
        eager = rt.add_adapters(buf.clone(), xd, w, slots)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf.view(torch.int16), eager.view(torch.int16))
        check(buf, nout, nx, nw, slots.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank", [72, 256])
def test_group_captured_first(rt, rank, dtype):
    """A group with operands past 64 KB of LDS, captured before any eager call of its kind, replayed on buffers
    that eager calls on the same workspace use in between."""
    rows, outputs = 70, (96, 33)
    cases = [host_case(rows, 200, n, rank, 3, dtype, 83 + n) for n in outputs]
    x, slots = cases[0][0], slots_of(rows, 3, 83)
    ws_of, xd, sl = [on_gpu(rt, c[1]) for c in cases], x.cuda(), slots.cuda()
    outs = [c[2].cuda() for c in cases]
    ws = torch.zeros(rt.adapters_workspace_bytes(ws_of, rows), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rt.add_adapters_group(outs, xd, ws_of, sl, workspace=ws)
    for _ in range(3):
        for o, c in zip(outs, cases):
            o.copy_(c[2])
        rt.add_adapters(torch.zeros(5, outputs[1], dtype=dtype, device="cuda"), xd, ws_of[1], sl, rows=5, workspace=ws)
        g.replay()
        torch.cuda.synchronize()
        for o, c in zip(outs, cases):
            check(o, c[2], x, c[1], slots)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rank,count", [(16, 40), (48, 40), (48, 3)])
def test_many_adapters_a_workgroup(rt, rank, count, dtype):
    """More adapters in a chunk than workgroups take them one each: the next one's operands do not meet the
    last one's sums."""
    rows = 4000
    case = host_case(rows, 96, 80, rank, count, dtype, 85)
    slots = slots_of(rows, count, 85)
    first = run(rt, case, slots)
    for _ in range(3):
        again = run(rt, case, slots)
        assert torch.equal(again, first)


def test_row_strides_past_every_product(rt):
    """A single row: its stride can be anything that 63 bits hold, and is not multiplied by a chunk's 64 rows."""
    case = host_case(1, 64, 48, 16, 2, torch.float32, 86)
    x, adapters, out = case
    slots = torch.tensor([1], dtype=torch.int32)
    for stride in (1 << 56, 1 << 57, 1 << 58):
        got = out.cuda()
        rt.add_adapters(got.as_strided((1, 48), (stride, 1)), x.cuda().as_strided((1, 64), (stride, 1)), on_gpu(rt, adapters),
                        slots.cuda())
        check(got, out, x, adapters, slots)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_repeatable(rt, rows):
    x, adapters, out = host_case(rows, 1280, 264, 32, 4, torch.float32, 81)
    w, xd, slots = on_gpu(rt, adapters), x.cuda(), slots_of(rows, 4, 81).cuda()
    first = rt.add_adapters(out.cuda(), xd, w, slots)
    for _ in range(3):
        assert torch.equal(rt.add_adapters(out.cuda(), xd, w, slots).view(torch.int32), first.view(torch.int32))


def test_beside_gguf_and_q4_projections(rt):
    """Onto the output of a shared projection of each weight kind, which is what the operator is for."""
    import numpy as np

    import oracle
    from qcheck import Q4Case
    q4 = Q4Case(256, 512, seed=91)
    native = oracle.q45k_random_native(256, 512, seed=92)
    w5 = rt.q5k_repack(torch.from_numpy(np.ascontiguousarray(native)).cuda(), 256, 512)
    x, adapters, _ = host_case(20, 512, 256, 16, 4, torch.float32, 93)
    slots = slots_of(20, 4, 93)
    for weight in (q4.w_tiled, q4.w_rm, w5):
        base = rt.gemm(weight, x.cuda(), out_dtype=torch.float32)
        before = base.cpu()
        rt.add_adapters(base, x.cuda(), on_gpu(rt, adapters), slots.cuda())
        check(base, before, x, adapters, slots)


def test_python_refusals(rt):
    from splosh_amd._lib import SploshError
    x, adapters, out = host_case(4, 64, 48, 8, 3, torch.float32, 1)
    w, xd, od = on_gpu(rt, adapters), x.cuda(), out.cuda()
    slots = slots_of(4, 3, 1).cuda()

    def refused(case, *args, **kw):
        with pytest.raises(SploshError) as e:
            rt.add_adapters(*args, **kw)
        assert e.value.case == case, e.value

    refused("unsupported", od, xd.float(), w, slots)
    refused("unsupported", od.half(), xd, w, slots)
    refused("unsupported", od.t(), xd, w, slots)
    refused("unsupported", od, xd, w, slots.long())
    refused("bufferTooSmall", od, xd, w, slots[:3])
    refused("unsupported", od, xd, w, slots.cpu())
    refused("nullPointer", od.cpu(), xd, w, slots)
    refused("nullPointer", od, xd.cpu(), w, slots)
    refused("bufferTooSmall", od, xd, w, torch.zeros(5, dtype=torch.int32, device="cuda"), rows=5)
    refused("invalidShape", od[:, :40].contiguous(), xd, w, slots)
    refused("invalidShape", od[:, :40], xd, w, slots)
    refused("invalidShape", od, xd[:, :63], w, slots)
    refused("bufferTooSmall", od[:3], xd, w, slots)
    refused("invalidShape", od, xd[:0], w, slots)
    refused("workspaceTooSmall", od, xd, w, slots, workspace=torch.zeros(16384, dtype=torch.uint8, device="cuda"))
    with pytest.raises(SploshError):
        rt.add_adapters_group([od, od], xd, [w, w], slots)
    with pytest.raises(SploshError):
        rt.add_adapters_group([od], xd, [w, w], slots)
    a, b = w.a, w.b
    for bad in ((a.float(), b), (a[0], b), (a[:2], b), (a, b.transpose(1, 2)), (a[:, :4], b), (a.cpu(), b.cpu()), (a, b.cpu()),
                (a, b, w.scales[:2]), (a, b, w.scales.double()), (a, b, w.scales, torch.zeros(3, device="cuda"))):
        with pytest.raises(SploshError):
            rt.Adapters(*bad)
    assert torch.equal(od.cpu(), out)
