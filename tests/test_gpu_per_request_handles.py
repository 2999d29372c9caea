"""The per-request operators' handles and workspaces on the device: what is refused leaves every output as it was."""
import pytest
import torch

from adapter_check import check
from test_gpu_adapters import host_case, on_gpu, slots_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from splosh_amd import runtime
    return runtime


def test_workspaces_on_the_host(rt):
    from splosh_amd._lib import SploshError
    x, adapters, out = host_case(4, 64, 48, 8, 3, torch.float32, 1)
    w, xd, od, slots = on_gpu(rt, adapters), x.cuda(), out.cuda(), slots_of(4, 3, 1).cuda()
    logits = torch.randn(4, 100).cuda()
    tokens = torch.full((4,), 7, dtype=torch.int32, device="cuda")
    far = torch.zeros(1 << 22, dtype=torch.uint8)
    one = torch.zeros(1, dtype=torch.uint8, device="cuda").expand(1 << 22)
    for ws in (far, one):
        for call in (lambda: rt.add_adapters(od, xd, w, slots, workspace=ws),
                     lambda: rt.add_adapters_group([od], xd, [w], slots, workspace=ws),
                     lambda: rt.sample(logits, out=tokens, workspace=ws)):
            with pytest.raises(SploshError) as e:
                call()
            assert e.value.case == "unsupported"
    assert torch.equal(od.cpu(), out) and (tokens == 7).all()


def test_adapters_keep_their_tensors(rt):
    """A handle holds the addresses of the tensors that it was made from: none can be put in their place, and
    writing into them is seen by the next call."""
    x, adapters, out = host_case(6, 64, 48, 8, 3, torch.float32, 2)
    w, slots = on_gpu(rt, adapters), slots_of(6, 3, 2)
    for name in ("a", "b", "scales", "ranks"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name))
    other = host_case(6, 64, 48, 8, 3, torch.float32, 3)[1]
    for mine, new in zip((w.a, w.b, w.scales), other):
        mine.copy_(new)
    got = out.cuda()
    rt.add_adapters(got, x.cuda(), w, slots.cuda())
    check(got, out, x, other, slots)
