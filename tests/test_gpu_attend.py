"""splosh_attend against its definition in 64 bits, over what the cache holds."""
import math

import pytest
import torch

from step_check import attended, check_bf16, kept, packed, places

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


class Step:
    """A cache filled for requests of given lengths, in 64 bits on the host and on the GPU, and a step's queries."""

    def __init__(self, rt, runs, lengths, q_heads, heads, dim, page, seed=0, shared=0, more=0, spread=1.0, pad=0, layout="dense"):
        gen = torch.Generator().manual_seed(seed)
        self.rt, self.runs, self.shared, self.page, self.dim = rt, runs, shared, page, dim
        self.starts, self.lengths, self.table, self.pages = packed(runs, lengths, page, seed, shared=shared, pad=pad)
        shape = (self.pages * page, heads, dim)
        size = torch.exp(spread * torch.randn(*shape[:2], 1, generator=gen))
        self.k = (torch.randn(*shape, generator=gen) * size).to(torch.bfloat16)
        self.v = (torch.randn(*shape, generator=gen) * size.flip(0)).to(torch.bfloat16)
        self.rows = sum(runs) + more
        wide = torch.randn(self.rows, q_heads, 2 * dim if layout == "gated" else dim, generator=gen).to(torch.bfloat16)
        self.q = wide[..., :dim]
        self.q_gpu = wide.cuda()[..., :dim]
        self.cache = rt.Cache.empty(self.pages, page, heads, dim, "cuda")
        self.fill()
        base = (self.table._base if self.table._base is not None else self.table).cuda()
        self.packed = rt.Packed(self.starts.cuda(), self.lengths.cuda(), base[:, : self.table.shape[1]])

    def fill(self):
        count = self.pages * self.page
        whole = torch.arange(self.pages, dtype=torch.int32).cuda()[None]
        ends = torch.tensor([0, count], dtype=torch.int32).cuda()
        self.rt.cache_write(self.cache, self.rt.Packed(ends, ends[1:].clone(), whole), self.k.cuda(), self.v.cuda())
        self.k64, self.v64 = ((lambda c: c[0] * c[1])(kept(t)) for t in (self.k, self.v))

    def run(self, **kw):
        out = torch.full((self.rows, self.q.shape[1], self.dim), 9.0, dtype=torch.bfloat16, device="cuda")
        return self.rt.attend(self.q_gpu, self.cache, self.packed, shared=self.shared, out=out, **kw)

    def want(self, scale=None):
        """[(rows, out, bound)] by request."""
        got = []
        for r, n in enumerate(self.runs):
            if n == 0:
                continue
            begin, length = int(self.starts[r]), int(self.lengths[r])
            table = self.table[r].long().clamp(min=0).clone()
            table[: self.shared // self.page] = self.table[0, : self.shared // self.page].long()
            slots = (table[:, None] * self.page + torch.arange(self.page)).flatten()[: max(length, 1)]
            position = length - n + torch.arange(n)
            out, off = attended(self.q[begin : begin + n], self.k64[slots], self.v64[slots], position, scale or self.dim ** -0.5)
            got.append((slice(begin, begin + n), out, off))
        return got

    def check(self, got, scale=None):
        got = got.cpu()
        for rows, out, off in self.want(scale):
            check_bf16(got[rows], out, off, f"rows {rows.start}..{rows.stop}")
        assert bool((got[sum(self.runs):] == 9).all())


@pytest.mark.parametrize("runs,lengths,q_heads,heads,dim,page", [
    ([1], [1], 1, 1, 64, 32), ([1], [31], 4, 2, 128, 32), ([1], [33], 24, 4, 256, 64), ([1], [700], 6, 1, 256, 96),
    ([1] * 5, [1, 32, 64, 65, 500], 8, 2, 128, 32), ([8] * 4, [8, 40, 129, 1000], 10, 2, 256, 256), ([11] * 3, [300, 40, 11], 5, 1, 256, 64), ([3, 0, 7, 1], [10, 77, 7, 333], 10, 2, 128, 96),
    ([5], [5], 7, 7, 64, 32), ([2, 9], [300, 41], 32, 1, 64, 64), ([40], [40], 6, 1, 256, 64), ([100, 3], [150, 9], 5, 1, 128, 32),
    ([333], [400], 8, 2, 64, 64), ([300], [1000], 6, 1, 256, 256), ([64, 64, 64], [64, 200, 65], 4, 4, 128, 32),
    ([700, 1, 2], [700, 2000, 2], 4, 1, 128, 96), ([200, 70], [1500, 70], 6, 1, 64, 96), ([130], [900], 4, 2, 64, 32), ([513], [513], 3, 3, 256, 32), ([1] * 300, [1 + 7 * i % 190 for i in range(300)], 4, 2, 64, 32)])
def test_attend(rt, runs, lengths, q_heads, heads, dim, page):
    s = Step(rt, runs, lengths, q_heads, heads, dim, page, seed=len(runs) + dim, more=2, layout="gated" if dim == 128 else "dense", pad=3)
    s.check(s.run())


@pytest.mark.parametrize("runs,own,shared,q_heads,heads,dim,page", [
    ([1, 1, 1], [5, 1, 40], 64, 4, 2, 128, 32), ([4] * 6, [4, 30, 64, 5, 100, 4], 512, 6, 1, 256, 256), ([3, 0, 2], [3, 9, 200], 96, 8, 2, 64, 96),
    ([40] * 5, [40, 41, 80, 333, 64], 1024, 6, 2, 128, 64), ([50, 50], [50, 70], 96, 4, 2, 64, 96), ([60, 9], [60, 70], 160, 4, 1, 128, 32), ([1] * 70, [1 + i for i in range(70)], 256, 2, 1, 256, 32)])
def test_shared_prefix(rt, runs, own, shared, q_heads, heads, dim, page):
    """The same as without saying so, to the bounds of both; and other requests' entries for it are not used."""
    s = Step(rt, runs, [shared + n for n in own], q_heads, heads, dim, page, seed=dim, shared=shared, more=1)
    s.check(s.run())
    s.packed.table[1:, : shared // page] = -5
    s.check(s.run())


def test_prefix_longer_than_a_request(rt):
    """A request whose rows lie inside the shared prefix sees it up to its own positions."""
    s = Step(rt, [3, 2, 4], [160 + 30, 50, 128], 4, 2, 128, 32, seed=4, shared=128)
    s.check(s.run())


@pytest.mark.parametrize("seed", range(24))
def test_any_step(rt, seed):
    """Steps of any shape: requests with no, one and many rows, groups of one to fifteen, pages of 32 to 1024 tokens, with and
    without a shared prefix, and rows before the first request and behind the last."""
    gen = torch.Generator().manual_seed(500 + seed)
    pick = lambda *v: v[int(torch.randint(0, len(v), (1,), generator=gen))]  # noqa: E731
    dim, heads, page, requests = pick(64, 128, 256), pick(1, 2, 3), pick(32, 64, 96, 1024), pick(1, 2, 5, 9, 67)
    group = pick(1, 2, 3, 5, 7, 15)
    shared = pick(0, 0, 1, 3) * page if page < 1024 else 0
    runs = [pick(0, 1, 1, 2, 4, 7) if requests > 2 else pick(1, 9, 33, 150) for _ in range(requests)]
    runs[-1] = max(runs[-1], 1)
    lengths = [shared + n + pick(0, 0, 1, 31, 100, 333) for n in runs]
    s = Step(rt, runs, lengths, heads * group, heads, dim, page, seed=seed, shared=shared, more=pick(0, 3), layout=pick("dense", "gated"),
             pad=pick(0, 1))
    scale = pick(None, 0.3)
    s.check(s.run(scale=scale), scale)


def test_rows_before_the_first_request(rt):
    """starts[0] above zero: those rows belong to no request."""
    s = Step(rt, [3, 50], [40, 90], 4, 2, 64, 32, seed=16)
    want = s.run()
    s.packed.starts[0] = 2
    for shared in (0, 32):
        got = rt.attend(s.q_gpu, s.cache, s.packed, shared=shared, out=torch.full_like(want, 9.0))
        assert bool((got[:2] == 9).all())
        if shared == 0:  # (request 0 has one row of the same position)
            assert torch.equal(got[2:], want[2:])


def test_lengths_past_the_table(rt):
    """A length of more tokens than the table has pages for: its rows see those that are there."""
    for rows in (2, 90):
        s = Step(rt, [rows], [96], 4, 2, 128, 32, seed=17)
        s.packed.lengths[0] = 96 + 1000
        slots = (s.table[0].long()[:, None] * 32 + torch.arange(32)).flatten()
        out, off = attended(s.q, s.k64[slots], s.v64[slots], torch.full((rows,), 95), 128 ** -0.5)
        check_bf16(s.run().cpu(), out, off)


def test_scales_far_apart(rt):
    """Values whose sizes differ by orders of magnitude, among them vectors of zeros, and sharp and flat weights."""
    for spread, scale in ((4.0, 0.01), (2.0, 3.0)):
        s = Step(rt, [4, 1], [300, 77], 4, 2, 128, 32, seed=6, spread=spread)
        s.v[::3] = 0
        s.fill()
        s.check(s.run(scale=scale), scale)


def test_rows_without_keys(rt):
    """Lengths of zero and shorter than their run: zeros. Pages that are none: masked; a row with nothing else: zeros."""
    s = Step(rt, [2, 3, 1, 4], [0, 2, 70, 4], 6, 2, 128, 32, seed=8)
    got = s.run().cpu()
    assert not got[:2].any() and not got[2].any()
    s.check(got)
    table = s.packed.table
    table[2, 0], table[3, 0] = s.pages, -1  # tokens 0..31 of request 2, all of request 3
    got = s.run().cpu()
    assert not got[6:].any()
    slots = (s.table[2, 1:].long()[:, None] * 32 + torch.arange(32)).flatten()[: 70 - 32]
    out, off = attended(s.q[5:6], s.k64[slots], s.v64[slots], torch.tensor([70 - 33]), 128 ** -0.5)
    check_bf16(got[5:6], out, off)


@pytest.mark.parametrize("rows,length,dim,page", [(3, 700, 128, 32), (100, 700, 64, 32), (100, 700, 128, 32), (90, 500, 256, 32), (130, 900, 64, 96)])
def test_holes_between_pages(rt, rows, length, dim, page):
    """Pages that are none, alone and side by side, first and last, below every kind of tile: their keys are masked."""
    s = Step(rt, [rows], [length], 2, 1, dim, page, seed=15)
    columns = -(-length // page)
    none = sorted({0, 2, 3, 4, 7, columns - 3, columns - 1})
    for i, column in enumerate(none):
        s.packed.table[0, column] = (-1, s.pages, -(2 ** 31), 2 ** 31 - 1)[i % 4]
    seen = torch.tensor([i // page not in none for i in range(length)])
    slots = (s.table[0].long()[:, None] * page + torch.arange(page)).flatten()[:length][seen]
    position = seen.long().cumsum(0)[length - rows + torch.arange(rows)] - 1
    out, off = attended(s.q, s.k64[slots], s.v64[slots], position, dim ** -0.5)
    check_bf16(s.run().cpu(), out, off)


@pytest.mark.parametrize("runs,lengths,dim", [([1], [50], 256), ([4, 8], [37, 65], 128), ([200], [230], 256), ([150], [230], 64)])
def test_what_is_masked_does_not_count(rt, runs, lengths, dim):
    """Infinities and NaN kept in the cache at masked tokens (behind each row, in pages of others, past the lengths) change nothing;
    at seen ones they make their own rows NaN."""
    s = Step(rt, runs, lengths, 4, 2, dim, 32, seed=9)
    clean = s.run()
    last = int(s.lengths[0]) - 1
    bad = int(s.table[0, last // 32]) * 32 + last % 32
    used = set()
    for r, n in enumerate(lengths):
        used |= {int(s.table[r, i // 32]) * 32 + i % 32 for i in range(n)}
    for slot in range(s.pages * 32):
        if slot not in used:
            s.k[slot], s.v[slot, :, 3] = math.inf, math.nan
    s.v[bad] = math.nan
    s.fill()
    got = s.run()
    sees = runs[0] - 1
    assert torch.isnan(got[sees]).all()
    rest = [m for m in range(s.rows) if m != sees]
    assert torch.equal(got[rest], clean[rest])
    # (bytes that were never written may be anything at all)
    s.v[bad] = 0
    s.fill()
    for slot in range(s.pages * 32):
        if slot not in used:
            record = s.cache.data[slot // 32].view(2, -1)
            record[:, slot % 32 * dim : (slot % 32 + 1) * dim] = 0x00
            scales = record[:, 64 * dim :].view(torch.float32)
            scales[:, slot % 32], scales[:, 32 + slot % 32] = -math.inf, [0.0, -1.0, math.inf, math.nan][slot % 4]
    s.check(s.run())


def test_queries_that_are_not_finite(rt):
    s = Step(rt, [3, 40], [70, 90], 4, 2, 128, 32, seed=10)
    clean = s.run()
    s.q_gpu[1, 2, 5], s.q_gpu[20, 0, 0] = math.nan, math.inf
    got = s.run()
    assert torch.isnan(got[1, 2]).all() and torch.isnan(got[20, 0]).any()
    same = torch.ones(s.rows, 4, dtype=torch.bool)
    same[1, 2] = same[20, 0] = False
    assert torch.equal(got[same.cuda()], clean[same.cuda()])


def test_queries_of_any_size(rt):
    """Queries near the ends of bf16 with scales that make up for it."""
    for size in (1e-36, 1e30):
        s = Step(rt, [2, 30], [70, 90], 4, 2, 64, 32, seed=11)
        s.q_gpu.copy_((s.q.float() * size).to(torch.bfloat16))
        s.q = s.q_gpu.cpu()
        s.check(s.run(scale=0.125 / size), 0.125 / size)


def test_the_same_again(rt):
    """Bit for bit: again, on another stream, with a workspace of garbage, and from a captured call whose lengths change."""
    s = Step(rt, [6, 1, 9], [800, 33, 9], 12, 2, 128, 64, seed=12)
    first = s.run()
    need = rt.attend_workspace_bytes(s.cache, s.packed, s.rows, 12)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    assert torch.equal(s.run(workspace=ws), first) and bool((ws[:16384] == 0xff).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = rt.attend(s.q_gpu, s.cache, s.packed, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(first)
    with torch.cuda.graph(g):
        rt.attend(s.q_gpu, s.cache, s.packed, out=out, workspace=ws)
    for lengths in ([800, 33, 9], [100, 1, 64], [800, 2, 10]):
        s.packed.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = s.run()
        torch.cuda.synchronize()
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), lengths


def test_far_pages(rt):
    """Pages past 4 GiB of the cache."""
    page, heads, dim = 256, 8, 256
    data = torch.zeros(4200, rt.cache_page_bytes(heads, dim, page), dtype=torch.uint8, device="cuda")
    cache = rt.Cache(data, page, heads, dim)
    table = torch.tensor([[4199, 4100, 3]], dtype=torch.int32)
    n = 600
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, heads, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(n, 16, dim, generator=gen).to(torch.bfloat16)
    ends, lengths = torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    p = rt.Packed(ends, lengths, table.cuda())
    rt.cache_write(cache, p, k.cuda(), v.cuda())
    for rows in (2, n):
        step = rt.Packed(torch.tensor([0, rows], dtype=torch.int32).cuda(), lengths, table.cuda())
        got = rt.attend(q[-rows:].cuda(), cache, step).cpu()
        (kc, ks), (vc, vs) = kept(k), kept(v)
        some = torch.arange(n - rows, n)
        out, off = attended(q[-rows:], kc * ks, vc * vs, some, dim ** -0.5)
        check_bf16(got, out, off)


def test_in_place(rt):
    """The output in its queries' place: written by one piece, joined from several, and with a shared prefix."""
    for runs, lengths, shared in (([2, 5], [900, 30], 0), ([300], [900], 0), ([4, 4], [140, 200], 128)):
        s = Step(rt, runs, lengths, 6, 2, 128, 32, seed=14, shared=shared)
        want = s.run()
        got = rt.attend(s.q_gpu, s.cache, s.packed, shared=shared, out=s.q_gpu)
        assert got.data_ptr() == s.q_gpu.data_ptr() and torch.equal(got, want)
