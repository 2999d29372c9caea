"""splosh_verify with draws at the end of the weight."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [100, 5000, 32003, 100003])
@pytest.mark.parametrize("spread,temperature", [(2.0, 0.1), (4.0, 0.2), (1.0, 1.0)])
def test_u_of_one_and_more(rt, dtype, vocab, spread, temperature):
    """u >= 1: the last entry with weight, however little of it: of p after a whole run, and of what a lookup's rejected token leaves."""
    rows, gen = 40, torch.Generator().manual_seed(vocab)
    x = (spread * torch.randn(2 * rows, vocab, generator=gen)).to(dtype)
    last = torch.randint(0, min(vocab, 700), (2 * rows,), generator=gen)
    last[::3] = 0
    x[torch.arange(vocab)[None] >= vocab - last[:, None]] = -float("inf")  # (masked behind the last entry)
    # No weight vanishes: (max - min) / T / ln 2 is below the 1022 powers of two of a 64-bit number.
    finite = x.double().masked_fill(x == -float("inf"), 0.0)
    assert float((x.double().amax(1) - finite.amin(1)).max()) / temperature * 1.4427 < 1000
    t = torch.full((2 * rows,), temperature)
    # Requests of one row, and of two whose drafted token, one without weight, is not accepted.
    for runs in (1, 2):
        requests = 2 * rows // runs
        starts = torch.arange(0, 2 * rows + 1, runs, dtype=torch.int32)
        tokens = torch.full((2 * rows,), -1, dtype=torch.int32)
        u = torch.tensor([1.0, 1.5, float("inf"), 1.0 + 2.0 ** -23]).repeat(rows // 2)
        got, accepted = rt.verify(x.cuda(), tokens.cuda(), starts.cuda(), u.cuda(), t[:requests].cuda())
        assert not accepted.any()
        assert torch.equal(got.cpu()[::runs].long(), (vocab - 1 - last)[::runs]), runs
