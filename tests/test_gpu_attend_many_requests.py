"""splosh_attend where its work is found by other ways than for small steps: more than 64 requests of many vectors each, and prompts of more than 64 tiles."""
import pytest
import torch

from step_check import attended, check_bf16
from test_gpu_attend import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


@pytest.mark.parametrize("dim,page,shared", [(64, 32, 0), (128, 64, 0), (256, 32, 0), (64, 64, 128), (128, 32, 96)])
def test_many_requests_of_many_vectors(rt, dim, page, shared):
    """70 requests that average more than 64 vectors, some without rows, one much longer than the others."""
    runs = [(11 * i) % 40 for i in range(70)]
    runs[33] = 300
    s = Step(rt, runs, [shared + n + (37 * i) % 150 for i, n in enumerate(runs)], 4, 1, dim, page, seed=dim, shared=shared, more=3)
    assert sum(runs) * 4 / 70 > 64
    s.check(s.run())


def test_a_long_prompt_among_many_requests(rt):
    """66 requests, one of them a prompt of more than 64 tiles."""
    runs = [1] * 66
    runs[40] = 2200
    s = Step(rt, runs, [n + (31 * i) % 90 for i, n in enumerate(runs)], 8, 1, 64, 32, seed=5)
    s.check(s.run())


@pytest.mark.parametrize("rows,past,q_heads,dim", [(2100, 0, 8, 64), (2100, 100, 8, 128), (1100, 33, 16, 256), (66 * 16 + 5, 400, 16, 64)])
@pytest.mark.parametrize("shared", [0, 64])
def test_prompts_of_more_than_64_tiles(rt, rows, past, q_heads, dim, shared):
    """Prompts of 256 vectors a tile, alone and beside a request of one row; rows checked where tiles begin and end, and some others."""
    s = Step(rt, [rows, 1], [shared + rows + past, shared + 77], q_heads, 1, dim, 64, seed=rows, shared=shared)
    assert rows * q_heads > 64 * 256
    got = s.run().cpu()
    for r, n in enumerate(s.runs):
        begin, length = int(s.starts[r]), int(s.lengths[r])
        pick = sorted({0, 1, n // 3, n // 2, n - 2, n - 1} | {m for t in (1, 31, 32, 63, 64, 65) for m in (256 * t // q_heads - 1, 256 * t // q_heads)})
        m = torch.tensor([i for i in pick if 0 <= i < n])
        table = s.table[r].long().clamp(min=0)
        slots = (table[:, None] * s.page + torch.arange(s.page)).flatten()[:length]
        out, off = attended(s.q[begin + m], s.k64[slots], s.v64[slots], length - n + m, dim ** -0.5)
        check_bf16(got[begin + m], out, off, f"request {r}")
