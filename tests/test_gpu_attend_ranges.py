"""splosh_attend at the ends of its numbers: values whose sizes lie as far apart as the cache can hold them, and scores near the ends of
fp32."""
import pytest
import torch

from step_check import HALF, attended, check_bf16
from test_gpu_attend import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


# few vectors and many, one record, one wave's and all waves', a segment cut over workgroups, each kind of join, and a shared prefix
SHAPES = [([1], [2], 1, 1, 64, 32, 0), ([1, 3], [70, 300], 2, 1, 128, 32, 0), ([1], [1500], 3, 1, 256, 96, 0), ([20], [700], 2, 1, 64, 64, 0), ([2, 2], [3000, 40], 6, 2, 128, 32, 0),
          ([4] * 150, [40] * 150, 8, 2, 128, 32, 0), ([600], [640], 8, 1, 64, 64, 0), ([700], [800], 6, 1, 256, 32, 0),
          ([90], [200], 1, 1, 256, 32, 0), ([100, 80], [1000, 80], 2, 1, 128, 32, 0), ([300], [400], 1, 1, 64, 96, 0), ([700], [900], 8, 1, 128, 64, 0),
          ([1, 2, 1], [300, 220, 290], 4, 2, 128, 32, 192), ([40, 60], [300, 700], 2, 1, 256, 32, 256), ([50, 70], [230, 200], 2, 1, 64, 96, 96)]


@pytest.mark.parametrize("order", ["by turns", "small first", "large first", "one small"])
@pytest.mark.parametrize("small,large", [(0.0, 1e10), (0.0, 1e30), (0.0, 3e38), (1e-27, 1e4), (1e-20, 1e25)])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_of_any_size(rt, shape, small, large, order):
    """Every key has its weight, whatever the size of its value: a value of zeros beside one of 1e30 leaves half of it, in one record,
    in two, in two pieces and in a prefix and behind it.

    The bound is step_check's: an exponent is a logarithm of a scale (up to 2^7, 2^-17 for its last place) and two roundings of sums of that
    size (2^-18 each), 2^-16 in all, beside the weights' 2^-11 and the output's 2^-8."""
    runs, lengths, q_heads, heads, dim, page, shared = shape
    s = Step(rt, runs, lengths, q_heads, heads, dim, page, seed=dim + len(order), shared=shared)
    unit = s.v.double() / s.v.double().abs().amax(-1, keepdim=True)
    for r, length in enumerate(lengths):
        i = torch.arange(length)
        slots = s.table[r].long()[i // page] * page + i % page
        pick = {"by turns": i % 2 == 1, "small first": i >= length // 2, "large first": i < length // 2, "one small": i != length // 3}[order]
        size = torch.where(pick, large, small).double()
        s.v[slots] = (unit[slots] * size[:, None, None]).to(torch.bfloat16)
    s.fill()
    s.check(s.run(scale=0.01), 0.01)


@pytest.mark.parametrize("runs,lengths,shared", [([1, 2], [40, 9], 0), ([8], [900], 0), ([300], [420], 0), ([40, 30], [140, 200], 128)])
def test_in_place_and_again(rt, runs, lengths, shared):
    """Values far apart with the output in its queries' place, in a workspace of garbage, and behind a key that only later rows see."""
    s = Step(rt, runs, lengths, 4, 2, 128, 32, seed=2, shared=shared)
    s.v[::2] = 0
    for r, length in enumerate(lengths):
        s.v[int(s.table[r, (length - 1) // 32]) * 32 + (length - 1) % 32] = 1e30
    s.fill()
    want = s.run()
    s.check(want)
    ws = torch.full((rt.attend_workspace_bytes(s.cache, s.packed, s.rows, 4, shared),), 0xff, dtype=torch.uint8, device="cuda")
    assert torch.equal(s.run(workspace=ws), want)
    got = rt.attend(s.q_gpu, s.cache, s.packed, shared=shared, out=s.q_gpu, workspace=ws)
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows,length,dim,page", [(3, 700, 128, 32), (100, 700, 64, 32), (90, 500, 256, 64), (1000, 1100, 64, 32)])
@pytest.mark.parametrize("layout", ["dense", "gated"])
def test_far_apart_between_holes(rt, rows, length, dim, page, layout):
    """Values far apart with pages that are none between them, keys that are NaN behind all rows but the last, a table shorter than the length, and queries
    and outputs that are not aligned."""
    s = Step(rt, [rows], [length], 8, 2, dim, page, seed=15, layout=layout)
    columns = -(-length // page)
    none = sorted({0, 2, 3, columns - 3})
    for i, column in enumerate(none):
        s.packed.table[0, column] = (-1, s.pages, -(2 ** 31), 2 ** 31 - 1)[i]
    i = torch.arange(length)
    all_slots = s.table[0].long()[i // page] * page + i % page
    s.v[all_slots[::3]] = 0
    s.v[all_slots[1::5]] *= 1e12
    last = int(all_slots[-1])
    s.k[last] = float("nan")
    s.fill()
    seen = torch.tensor([j // page not in none for j in range(length)])
    seen[-1] = False
    slots = all_slots[seen]
    position = seen.long().cumsum(0)[length - rows + torch.arange(rows)] - 1
    out, off = attended(s.q, s.k64[slots], s.v64[slots], position, 0.01)
    got = s.run(scale=0.01)
    check_bf16(got[:-1].cpu(), out[:-1], off[:-1])
    assert torch.isnan(got[-1]).all()
    # One element off: no vector of q, and no row of the output, is where wide loads and stores could take it.
    wide = torch.zeros(rows, 8 * dim + 3, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 1 : 1 + 8 * dim].unflatten(1, (8, dim))
    q.copy_(s.q_gpu)
    held = torch.full((rows, 8 * dim + 3), 9.0, dtype=torch.bfloat16, device="cuda")
    rt.attend(q, s.cache, s.packed, scale=0.01, out=held[:, 1 : 1 + 8 * dim].unflatten(1, (8, dim)))
    same = held[:, 1 : 1 + 8 * dim].unflatten(1, (8, dim))
    assert torch.equal(same[:-1], got[:-1]) and torch.isnan(same[-1]).all()
    assert bool((held[:, :1] == 9).all()) and bool((held[:, 1 + 8 * dim :] == 9).all())


@pytest.mark.parametrize("runs,lengths,dim", [([3], [40], 64), ([2], [900], 128), ([1, 2], [300, 33], 256), ([80], [200], 64), ([90], [130], 128), ([150], [700], 256)])
def test_scores_of_any_size(rt, runs, lengths, dim):
    """Scores far below -1e30 and above 1e30: all of a row's weight is at its largest score, and the row is that key's value, to the rounding of
    its scale's reciprocal (2^-22) and the output's."""
    for sign in (-1.0, 1.0):
        s = Step(rt, runs, lengths, 2, 2, dim, 32, seed=3)
        s.q[:] = 1e17
        s.q_gpu.copy_(s.q)
        want = []
        for r, length in enumerate(lengths):
            i = torch.arange(length)
            slots = s.table[r].long()[i // 32] * 32 + i % 32
            # (The largest score is that of the row's first key or of its last one.)
            s.k[slots] = (sign * 1e17 * (1 + i / 64.0)).to(torch.bfloat16)[:, None, None].expand(-1, 2, dim)
            for m in range(runs[r]):
                want.append(int(slots[length - runs[r] + m if sign > 0 else 0]))
        s.fill()
        k = s.k64[torch.tensor(want)][:, :, 0]
        assert bool((k.abs() * 1e17 * dim * dim ** -0.5 > 1e34).all())
        got = s.run().cpu().double()
        for m, slot in enumerate(want):
            if sign > 0:  # (bf16 keys: neighbours of the last one may be equal to it)
                same = (s.k64[:, :, 0] == s.k64[slot, :, 0]).all(1).nonzero()[:, 0]
                if len(same) > 1:
                    continue
            v = s.v64[slot]
            assert bool(((got[m] - v).abs() <= v.abs() * (HALF + 2.0 ** -20)).all()), (sign, m)
