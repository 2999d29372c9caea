"""splosh_attend with starts that do not ascend: what a request's rows get is not defined, but nothing else changes, and the next call is right."""
import pytest
import torch

from test_gpu_attend import Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


@pytest.mark.parametrize("requests", [5, 64, 70, 300])
@pytest.mark.parametrize("rows", [1, 4, 40])
@pytest.mark.parametrize("shared", [0, 32])
def test_descending(rt, requests, rows, shared):
    s = Step(rt, [rows] * requests, [shared + rows + 3 * i % 50 for i in range(requests)], 4, 2, 64, 32, seed=requests, shared=shared)
    want = s.run()
    good = s.packed.starts.clone()
    gen = torch.Generator().manual_seed(requests)
    for turn in range(4):
        bad = good.cpu()[torch.randperm(requests + 1, generator=gen)] if turn < 2 else good.cpu().flip(0) if turn == 2 else \
            torch.where(torch.arange(requests + 1) % 2 == 0, 0, s.rows).to(torch.int32)
        s.packed.starts.copy_(bad)
        before = s.cache.data.clone()
        held = torch.full((s.rows + 64, 4, 64), 9.0, dtype=torch.bfloat16, device="cuda")
        rt.attend(s.q_gpu, s.cache, s.packed, shared=shared, out=held[32:-32])
        torch.cuda.synchronize()
        assert torch.equal(s.cache.data, before) and bool((held[:32] == 9).all()) and bool((held[-32:] == 9).all())
        s.packed.starts.copy_(good)
        assert torch.equal(s.run(), want)


@pytest.mark.parametrize("requests", [5, 70])
def test_outside_of_the_rows(rt, requests):
    """starts below 0 and past the call's rows, in any order, count as 0 and as the rows."""
    s = Step(rt, [0, 0] + [2] * (requests - 4) + [0, 0], [9] * requests, 4, 2, 64, 32, seed=3)
    want = s.run()
    s.packed.starts[0], s.packed.starts[1] = -3, -7
    s.packed.starts[-3:] = torch.tensor([s.rows + 9, s.rows + 900, s.rows + 5], dtype=torch.int32)
    assert torch.equal(s.run(), want)
