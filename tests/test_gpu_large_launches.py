"""The attention layers of steps so large that a launch has more than 2^32 threads."""
import pytest
import torch

from step_check import attended, check_bf16, kept

pytestmark = pytest.mark.gpu
ROWS, HEADS, DIM, PAGE = 1 << 22, 64, 64, 32  # (2^28 vectors of 64: 34 GB of bf16)


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


@pytest.fixture(autouse=True)
def returned():
    """The memory goes back to the device: the other tests' is small."""
    yield
    torch.cuda.empty_cache()


def step(rt, heads, seed):
    """A cache of one page, of one request whose last row is its token ROWS, so that all rows but the first 32 lie past the table."""
    gen = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(PAGE, heads, DIM, generator=gen).to(torch.bfloat16) for _ in range(2))
    cache = rt.Cache.empty(1, PAGE, heads, DIM, "cuda")
    ends, table = torch.tensor([0, PAGE], dtype=torch.int32).cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda()
    rt.cache_write(cache, rt.Packed(ends, ends[1:].clone(), table), k.cuda(), v.cuda())
    return cache, rt.Packed(torch.tensor([0, ROWS], dtype=torch.int32).cuda(), torch.tensor([ROWS], dtype=torch.int32).cuda(), table), k, v


def test_read(rt):
    cache, p, k, _ = step(rt, HEADS, 1)
    out = torch.empty(ROWS, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    for at in (0, 31, 32, ROWS // 2, ROWS - 2):
        out[at : at + 2] = 7.0
    rt.cache_read(cache, p, ROWS, k=out)
    codes, scales = kept(k)
    assert torch.equal(out[:PAGE].cpu(), (codes * scales).to(torch.bfloat16))
    for at in (32, ROWS // 2, ROWS - 2):
        assert not out[at : at + 2].any()


def test_attend(rt):
    cache, p, k, v = step(rt, 1, 2)
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(ROWS + HEADS, DIM, generator=gen).to(torch.bfloat16)
    q_gpu = q.cuda().as_strided((ROWS, HEADS, DIM), (DIM, DIM, 1))  # (vector (m, h) is number m + h)
    out = torch.empty(ROWS, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    rt.attend(q_gpu, cache, p, out=out)
    k64, v64 = ((lambda c: c[0] * c[1])(kept(t)) for t in (k, v))
    for at in (0, 30, 12345, ROWS // 2, ROWS - 3):
        m = at + torch.arange(3)
        vectors = q[m[:, None] + torch.arange(HEADS)]
        check_bf16(out[m.cuda()].cpu(), *attended(vectors, k64, v64, m.clamp(max=PAGE - 1), DIM ** -0.5), f"rows from {at}")
