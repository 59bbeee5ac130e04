"""Refusals of the expert linears' entry points (no GPU work is reached)."""
import os

import pytest
import torch


def test_python_refusals():
    from ictc_o3 import expert_linear, expert_order
    with pytest.raises(ValueError, match="device"):
        expert_order(torch.zeros(3, dtype=torch.int64), 2)
    with pytest.raises(TypeError, match="order"):
        expert_linear(torch.zeros(3, 4), torch.zeros(2, 4, 4), None)


def test_native_refusals():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")

    def rows(dtype=0, x=16, ldx=8, n=4, K=8, M=8, E=2, perm=16):
        nat.call("ictc_expert_linear", dtype, x, ldx, n, K, 16, None, M, E, perm, 16, 0, 16, None)

    for bad in (dict(dtype=4), dict(n=-1), dict(K=0), dict(M=0), dict(K=70000, ldx=70000), dict(E=0), dict(ldx=7),
                dict(x=None), dict(perm=None), dict(n=1 << 31)):
        with pytest.raises(ValueError):
            rows(**bad)
    rows(n=0, x=None)
    size = nat.lib().ictc_expert_outer_workspace_bytes
    assert size(0, 50, 8, 8, 2) == 0 and size(0, 100000, 8, 8, 2) > 0
    assert size(0, -1, 8, 8, 2) == -1 and size(7, 1, 8, 8, 2) == -1 and size(0, 1, 8, 0, 2) == -1
    with pytest.raises(ValueError, match="workspace"):
        nat.call("ictc_expert_outer", 0, 16, 8, 16, 8, 100000, 8, 8, 2, 16, 16, 16, None, 16, 8, None)
    with pytest.raises(ValueError):
        nat.call("ictc_expert_outer", 0, 16, 7, 16, 8, 4, 8, 8, 2, 16, 16, 16, None, None, 0, None)
