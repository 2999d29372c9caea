"""An output at its input's address is taken only where a vector's threads are alone with it: bf16, with the same strides (no GPU)."""
import ctypes

import pytest

from splosh_amd import _lib
from test_step_refusals import P, attend, heads, name, queries, write


@pytest.mark.parametrize("change", [dict(ld=1040), dict(row=2048), dict(head=256, row=2048), dict(head=256, row=2048, ld=2048)])
def test_attend(change):
    assert attend(q=P[5], out=P[5], ws_bytes=1, **change) == "layoutMismatch"
    assert attend(q=P[5], out=P[5], ws_bytes=1) == "workspaceTooSmall"  # (the same strides: nothing to refuse but the workspace)
    assert attend(q=P[5], out=P[5], ws_bytes=1, rows=1, row=4096) == "workspaceTooSmall"


@pytest.mark.parametrize("change", [dict(ld_out=1040), dict(row_stride=2048), dict(row_stride=2048, head_stride=256, ld_out=2048)])
def test_heads(change):
    part = queries(x=P[5], out=P[5], **change)
    assert write(q=part) == "layoutMismatch"
    listed = (_lib.Heads * 1)(part)
    rotate = lambda parts, dtype: name(_lib.lib().splosh_rotate_heads(ctypes.addressof(parts), 1, dtype, 5, 128, P[7], P[8], 64, 1e-6, None))  # noqa: E731
    assert rotate(listed, _lib.BF16) == "layoutMismatch"
    assert rotate((_lib.Heads * 1)(queries(x=P[5], out=P[5])), _lib.F32) == "layoutMismatch"


def test_cache_write_of_fp32():
    assert write(k=heads(), v=heads(), q=queries(x=P[5], out=P[5]), dtype=_lib.F32) == "layoutMismatch"
