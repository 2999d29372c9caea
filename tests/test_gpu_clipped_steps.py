"""A step's rows where `starts` pass the call's rows, and lengths at the ends of 32 bits: every operator of the attention layers has a row at
the same position, that of a step whose starts end at the call's rows."""
import pytest
import torch

from step_check import attended, check_bf16, kept, packed, places, rotated

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def filled(rt, heads, dim, page, pages, seed):
    """A cache with something in each place, in 64 bits on the host and on the GPU."""
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(pages * page, heads, dim, generator=gen).to(torch.bfloat16) for _ in range(2))
    cache = rt.Cache.empty(pages, page, heads, dim, "cuda")
    ends = torch.tensor([0, pages * page], dtype=torch.int32).cuda()
    rt.cache_write(cache, rt.Packed(ends, ends[1:].clone(), torch.arange(pages, dtype=torch.int32).cuda()[None]), k.cuda(), v.cuda())
    return cache, *((lambda c: c[0] * c[1])(kept(t)) for t in (k, v))


@pytest.mark.parametrize("starts,rows,lengths,shared", [
    ([0, 8], 4, [100], 64), ([0, 3, 20, 30], 7, [90, 130, 200], 64), ([0, 2, 90], 80, [70, 150], 0), ([0, 1, 200, 201, 300], 150, [65, 190, 70, 99], 64)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_starts_past_the_rows(rt, starts, rows, lengths, shared, dim):
    page, heads, group, half = 32, 2, 3, dim // 4
    runs = [max(0, min(b, rows) - min(a, rows)) for a, b in zip(starts, starts[1:])]
    ends, lengths_of, table, pages = packed(runs, lengths, page, 5, shared=shared)
    cache, k64, v64 = filled(rt, heads, dim, page, pages, 6)
    p = rt.Packed(torch.tensor(starts, dtype=torch.int32).cuda(), lengths_of.cuda(), table.cuda())
    at = places(ends.tolist(), lengths, table, page, pages, rows)
    gen = torch.Generator().manual_seed(7)
    k, v, q = (torch.randn(rows, n, dim, generator=gen).to(torch.bfloat16) for n in (heads, heads, heads * group))
    f = (1.0e4 ** (-torch.arange(half, dtype=torch.float64) / half)).float()

    # What lies at the rows' places is read ...
    slots = torch.tensor([place[2] * page + place[3] for place in at])
    for got, want in zip(rt.cache_read(cache, p, rows), (k64, v64)):
        assert torch.equal(got.cpu(), want[slots].to(torch.bfloat16))
    # ... and written, the queries turned by their positions, ...
    before = cache.data.clone()
    out = rt.cache_write(cache, p, k.cuda(), v.cuda(), q.cuda(), f.cuda())
    position = torch.tensor([place[1] for place in at])
    check_bf16(out.cpu(), *rotated(q, None, f, position, EPS), "q")
    whole = rt.Packed(ends.cuda(), lengths_of.cuda(), table.cuda())
    after = cache.data.clone()
    cache.data.copy_(before)
    rt.cache_write(cache, whole, k.cuda(), v.cuda(), q.cuda(), f.cuda())
    assert torch.equal(cache.data, after)
    # ... and seen up to them, also where a prefix is read apart from the rest.
    for common in {0, shared}:
        got = rt.attend(q.cuda(), cache, p, shared=common)
        assert torch.equal(got, rt.attend(q.cuda(), cache, whole, shared=common))
    cache.data.copy_(before)
    got = rt.attend(q.cuda(), cache, p, shared=shared).cpu()
    for r, n in enumerate(runs):
        if n:
            i = torch.arange(lengths[r])
            seen = table[r].long()[i // page] * page + i % page
            b = int(ends[r])
            check_bf16(got[b : b + n], *attended(q[b : b + n], k64[seen], v64[seen], lengths[r] - n + torch.arange(n), dim ** -0.5), f"request {r}")


@pytest.mark.parametrize("rows", [2, 70])
def test_lengths_at_their_ends(rt, rows):
    """Lengths next to -2^31: rows before the request's first token, which see nothing and are kept nowhere, of a shared prefix neither.
    Lengths next to 2^31: rows past the table, which see all of it."""
    page, dim = 32, 128
    table = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    cache, k64, v64 = filled(rt, 1, dim, page, 4, 8)
    q = torch.randn(rows, 2, dim, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    starts = torch.tensor([0, rows], dtype=torch.int32).cuda()
    for length in (-2 ** 31, -2 ** 31 + 1, -2 ** 31 + rows, -5, 2 ** 31 - 1):
        p = rt.Packed(starts, torch.tensor([length], dtype=torch.int32).cuda(), table.cuda())
        before = cache.data.clone()
        rt.cache_write(cache, p, q[:, :1].cuda(), q[:, 1:].cuda())
        assert torch.equal(cache.data, before)
        for got in rt.cache_read(cache, p, rows):
            assert not got.any()
        for shared in (0, 64, 128):
            got = rt.attend(q.cuda(), cache, p, shared=shared).cpu()
            if length < 0:
                assert not got.any(), (length, shared)
            else:
                check_bf16(got, *attended(q, k64, v64, torch.full((rows,), 127), dim ** -0.5), (length, shared))
