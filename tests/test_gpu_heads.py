"""splosh_rotate_heads, splosh_cache_write and splosh_cache_read against their definitions in 64 bits."""
import math

import pytest
import torch

from step_check import check_bf16, kept, packed, places, rotated

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
EPS = 1e-6


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def vectors(rows, heads, dim, dtype, seed, layout="dense"):
    gen = torch.Generator().manual_seed(seed)
    x = (1.5 * torch.randn(rows, heads, dim, generator=gen)).to(dtype)
    if layout == "dense":
        return x
    if layout == "gated":  # each head beside a gate
        wide = torch.full((rows, heads, 2 * dim), 7.0, dtype=dtype)
        wide[..., :dim] = x
        return wide[..., :dim]
    wide = torch.full((rows, heads * dim + 13), 7.0, dtype=dtype)  # odd rows, one element off
    wide[:, 1 : 1 + heads * dim] = x.reshape(rows, -1)
    return wide[:, 1 : 1 + heads * dim].unflatten(1, (heads, dim))


def on(t):
    """`t` on the GPU in the layout it has."""
    base = t if t._base is None else t._base
    return base.cuda().as_strided(t.shape, t.stride(), t.storage_offset())


def norm_weight(dim, seed):
    return (1 + 0.3 * torch.randn(dim, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16)


def frequencies_of(half, theta=1.0e7):
    return (theta ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,dim,rotary,layout", [
    (1, (24, 4), 256, 64, "gated"), (3, (5, 1), 256, 256, "dense"), (17, (6, 2), 128, 128, "odd"), (70, (3, 3, 1), 64, 64, "dense"),
    (2, (1,), 64, 2, "odd"), (5, (7, 2), 128, 42, "gated"), (9, (4,), 256, 0, "dense"), (1100, (2, 1), 128, 32, "dense")])
def test_rotate(rt, dtype, rows, heads, dim, rotary, layout):
    xs = [vectors(rows, n, dim, dtype, 10 + i, layout) for i, n in enumerate(heads)]
    weights = [norm_weight(dim, 20 + i) if i != 1 else None for i in range(len(heads))]
    positions = torch.randint(0, 1 << 20, (rows,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    positions[0] = 0
    f = frequencies_of(rotary // 2) if rotary else None
    outs = rt.rotate_heads([on(x) for x in xs], positions.cuda(), f.cuda() if rotary else None,
                           [w.cuda() if w is not None else None for w in weights], EPS)
    for i, (x, w, got) in enumerate(zip(xs, weights, outs)):
        want, off = rotated(x, w, f, positions, EPS)
        check_bf16(got.cpu(), want, off, f"part {i}")


def test_rotate_ends(rt):
    """Rows of zeros, of the largest and of the smallest values, far and negative positions, and rows in place."""
    x = torch.randn(6, 2, 128, generator=torch.Generator().manual_seed(1))
    x[0], x[1], x[2] = 0.0, x[1] * 1e18, x[2] * 1e-18
    x = x.to(torch.bfloat16)
    w, f = norm_weight(128, 2), frequencies_of(64, 1.0e4)
    positions = torch.tensor([5, 0, 1, 2 ** 31 - 1, -7, -2 ** 31], dtype=torch.int32)
    buffer = torch.full((6, 300), 3.0, dtype=torch.bfloat16, device="cuda")
    inside = buffer[:, 20:276].unflatten(1, (2, 128))
    inside.copy_(x)
    rt.rotate_heads([inside], positions.cuda(), f.cuda(), [w.cuda()], EPS, outs=[inside])
    want, off = rotated(x, w, f, positions, EPS)
    check_bf16(inside.cpu(), want, off)
    assert bool((buffer[:, :20] == 3).all()) and bool((buffer[:, 276:] == 3).all())


def written(rt, runs, lengths, heads, dim, page, dtype, seed, layout="dense", rotary=None, more=0, spare=2):
    """A written step: everything on the host, and the cache."""
    starts, lengths, table, pages = packed(runs, lengths, page, seed, spare)
    rows = sum(runs) + more
    k, v = vectors(rows, heads, dim, dtype, seed + 1, layout), vectors(rows, heads, dim, dtype, seed + 2, layout)
    q = vectors(rows, 3, dim, dtype, seed + 3, layout)
    f = frequencies_of(rotary // 2) if rotary else None
    kw, qw = (norm_weight(dim, seed + 4), norm_weight(dim, seed + 5)) if rotary else (None, None)
    cache = rt.Cache.empty(pages, page, heads, dim, "cuda")
    cache.data.fill_(0x5a)
    p = rt.Packed(starts.cuda(), lengths.cuda(), table.cuda())
    out = torch.full((rows, 3, dim), 9.0, dtype=torch.bfloat16, device="cuda")
    rt.cache_write(cache, p, on(k), on(v), on(q), *(t.cuda() if t is not None else None for t in (f, kw, qw)), EPS, out=out)
    return dict(starts=starts, lengths=lengths, table=table, pages=pages, rows=rows, k=k, v=v, q=q, f=f, kw=kw, qw=qw, cache=cache,
                packed=p, out=out.cpu(), at=places(starts.tolist(), lengths.tolist(), table, page, pages, rows))


CASES = [([1], [1], 2, 256, 32), ([8, 8, 8], [40, 8, 300], 4, 256, 256), ([1, 0, 5, 3], [97, 50, 5, 64], 2, 128, 96),
         ([33], [33], 1, 64, 32), ([2, 2], [65, 1], 2, 128, 32), ([70, 1], [70, 4000], 8, 64, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("runs,lengths,heads,dim,page", CASES)
def test_cache_holds_what_it_was_given(rt, dtype, runs, lengths, heads, dim, page):
    """Codes and scales of vectors kept as they are, read from the cache's bytes: exact, and nothing else is written."""
    st = written(rt, runs, lengths, heads, dim, page, dtype, 7, "odd", more=3)
    data = st["cache"].data.cpu()
    blocks, size = page // 32, 64 * dim + 256
    seen = torch.zeros_like(data, dtype=torch.bool)
    for m, place in enumerate(st["at"]):
        if place is None or place[1] < 0:
            continue
        for h in range(heads):
            base = (h * blocks + place[3] // 32) * size
            token = place[3] % 32
            for values, x in ((0, st["k"]), (1, st["v"])):
                codes, scale = kept(x[m, h])
                at = base + (values * 32 + token) * dim
                got = data[place[2], at : at + dim].int() - 128
                if dtype == torch.bfloat16:
                    assert torch.equal(got.double(), codes), (m, h, values)
                else:  # (x 127 / max, each rounded: a code next to the border of two can be either)
                    assert bool(((got.double() - x[m, h].double() * 127 / x[m, h].double().abs().max()).abs() <= 0.5 + 127 * 2 ** -23).all())
                seen[place[2], at : at + dim] = True
                at = base + 64 * dim + (values * 32 + token) * 4
                assert abs(float(data[place[2], at : at + 4].view(torch.float32)) / float(scale) - 1) <= 2 ** -24
                seen[place[2], at : at + 4] = True
    assert bool((data[~seen] == 0x5a).all())
    k, v = rt.cache_read(st["cache"], st["packed"], st["rows"])
    for got, x in ((k.cpu(), st["k"]), (v.cpu(), st["v"])):
        for m, place in enumerate(st["at"]):
            if place is None:
                continue
            x64 = x[m].double()
            step = x64.abs().amax(-1, keepdim=True) / 127
            d = (got[m].double() - (x64 if place[1] >= 0 else 0)).abs()
            assert bool((d <= step * (0.5 + 2 ** -14) + (x64.abs() + step) * 2 ** -8).all()), m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("runs,lengths,heads,dim,page,rotary", [c + (r,) for c, r in zip(CASES, (64, 256, 50, 64, 2, 32))])
def test_normed_and_turned(rt, dtype, runs, lengths, heads, dim, page, rotary):
    """The step's queries and keys by its rows' own positions; rows behind the last request left as they were."""
    st = written(rt, runs, lengths, heads, dim, page, dtype, 11, "gated", rotary, more=2)
    mine = torch.tensor([p is not None for p in st["at"]])
    position = torch.tensor([p[1] if p else 0 for p in st["at"]])
    want, off = rotated(st["q"], st["qw"], st["f"], position, EPS)
    check_bf16(st["out"][mine], want[mine], off[mine], "q")
    assert bool((st["out"][~mine] == 9).all())
    k, v = (t.cpu().double() for t in rt.cache_read(st["cache"], st["packed"], st["rows"]))
    want, off = rotated(st["k"], st["kw"], st["f"], position, EPS)
    for m, place in enumerate(st["at"]):
        if place is None:
            continue
        if place[1] < 0:
            assert not k[m].any() and not v[m].any()
            continue
        for got, x, o in ((k[m], want[m], off[m]), (v[m], st["v"][m].double(), torch.zeros(()))):
            # Half a step of 8 bits, the codes' own arithmetic, and the reading's rounding to bf16.
            step = (x.abs() + o).amax(-1, keepdim=True) / 127
            assert bool(((got - x).abs() <= (step * (0.5 + 2 ** -14) + 2 * o) * (1 + 2 ** -8) + x.abs() * 2 ** -8).all()), m


def test_cache_ends(rt):
    """Vectors of zeros, near the ends of fp32 and below the least scale, and ones that are not finite."""
    f32 = torch.float32
    x = torch.randn(10, 1, 64, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    for i, s in enumerate([0.0, 1e38, 3e-30, 1e-33, 1e-38, 1e-44]):
        x[i] *= s
    x = x.clamp(-3.4e38, 3.4e38).to(f32)
    x[1, 0, 3] = torch.finfo(f32).max
    x[7, 0, 5], x[8, 0, 6], x[9, 0, 7] = math.inf, -math.inf, math.nan
    starts, lengths, table, pages = packed([10], [10], 32)
    cache = rt.Cache.empty(pages, 32, 1, 64, "cuda")
    p = rt.Packed(starts.cuda(), lengths.cuda(), table.cuda())
    rt.cache_write(cache, p, x.cuda(), x.flip(0).cuda())
    k, v = (t.cpu() for t in rt.cache_read(cache, p, 10))
    for got, want in ((k, x), (v, x.flip(0))):
        for m in range(10):
            if not torch.isfinite(want[m]).all():
                assert torch.isnan(got[m]).all()
                continue
            step = max(float(want[m].double().abs().max()) / 127, 2.0 ** -100)
            # bf16 ends at 2^128 - 2^120: what is 2^128 - 2^119 or more, as fp32's largest, is read as infinite.
            over = want[m].double().abs() >= 2.0 ** 128 - 2.0 ** 119
            assert bool((got[m][over] == want[m][over].sign() * math.inf).all()), m
            # (fp32's own steps near its lower end, and the reading's rounding to bf16.)
            off = (got[m].double() - want[m].double()).abs()
            assert bool((off <= step * 0.51 + want[m].double().abs() * 2 ** -8 + 2.0 ** -133)[~over].all()), m


def test_pages_that_are_none(rt):
    """Page ids below 0 and past the cache, columns past the table, lengths shorter than their runs: nothing is
    written there, zeros are read, and every other row has its place."""
    page, dim = 32, 64
    starts = torch.tensor([0, 3, 6, 40, 41], dtype=torch.int32)
    lengths = torch.tensor([1, 70, 34, 65], dtype=torch.int32)  # (request 0: two rows before its first token)
    table = torch.tensor([[0, -1], [2, 5], [7, 1], [1 << 30, 3]], dtype=torch.int32)  # (5 pages; 70 > two pages)
    rows, pages = 41, 5
    k, v = vectors(rows, 2, dim, torch.bfloat16, 1), vectors(rows, 2, dim, torch.bfloat16, 2)
    cache = rt.Cache.empty(pages, page, 2, dim, "cuda")
    p = rt.Packed(starts.cuda(), lengths.cuda(), table.cuda())
    rt.cache_write(cache, p, k.cuda(), v.cuda())
    gk, gv = (t.cpu() for t in rt.cache_read(cache, p, rows))
    for m, place in enumerate(places(starts.tolist(), lengths.tolist(), table, page, pages, rows)):
        for got, x in ((gk, k), (gv, v)):
            if place[2] is None:
                assert not got[m].any(), m
            else:
                step = x[m].double().abs().amax(-1, keepdim=True) / 127
                assert bool(((got[m].double() - x[m].double()).abs() <= step * 0.51 + (x[m].double().abs() + step) * 2 ** -8).all()), m
    assert not cache.data[4].any()


def test_one_side_read(rt):
    st = written(rt, [4], [9], 2, 128, 32, torch.bfloat16, 3)
    k, v = rt.cache_read(st["cache"], st["packed"], 4)
    only = torch.full_like(v, 5.0)
    assert rt.cache_read(st["cache"], st["packed"], v=only) == (None, only) and torch.equal(only, v)
    only = torch.full_like(k, 5.0)
    rt.cache_read(st["cache"], st["packed"], k=only)
    assert torch.equal(only, k)


def test_far_pages(rt):
    """Pages past 4 GiB of the cache, and layers that lie beside each other in its pages."""
    page, heads, dim = 256, 8, 256
    size = 8 * 8 * (64 * 256 + 256)
    data = torch.empty(2200, 2 * size, dtype=torch.uint8, device="cuda")
    assert 2100 * 2 * size > 1 << 32
    starts, lengths = torch.tensor([0, 5], dtype=torch.int32), torch.tensor([259], dtype=torch.int32)
    table = torch.tensor([[2101, 2199]], dtype=torch.int32)
    p = rt.Packed(starts.cuda(), lengths.cuda(), table.cuda())
    kept_of = []
    for layer in range(2):
        cache = rt.Cache(data[:, layer * size : (layer + 1) * size], page, heads, dim)
        k, v = vectors(5, heads, dim, torch.bfloat16, 30 + layer), vectors(5, heads, dim, torch.bfloat16, 40 + layer)
        rt.cache_write(cache, p, k.cuda(), v.cuda())
        kept_of.append((cache, k, v))
    for cache, k, v in kept_of:
        for got, x in zip(rt.cache_read(cache, p, 5), (k, v)):
            step = x.double().abs().amax(-1, keepdim=True) / 127
            assert bool(((got.cpu().double() - x.double()).abs() <= step * 0.51 + (x.double().abs() + step) * 2 ** -8).all())
