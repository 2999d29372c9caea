"""What the Python entry points of the per-request operators refuse of a workspace (no GPU)."""
import pytest
import torch

from splosh_amd import runtime as rt
from splosh_amd._lib import SploshError


@pytest.mark.parametrize("workspace,index", [(torch.zeros(64), 0), (torch.zeros(64, dtype=torch.uint8).expand(4, 64), -1),
                                             (torch.zeros(64)[::2], -1), (torch.zeros(1).expand(1 << 20), -1)])
def test_workspaces(workspace, index):
    """On the host where the operands are on a device; views whose elements are fewer bytes than they seem."""
    with pytest.raises(SploshError) as e:
        rt._given_workspace(workspace, index)
    assert e.value.case == "unsupported"


def test_dense_workspace():
    ws = torch.zeros(10, 16, dtype=torch.int32)
    assert rt._given_workspace(ws[2:], -1) == (ws.data_ptr() + 128, 512)
