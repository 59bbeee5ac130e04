"""Refusals of the layer norm's entry points (no GPU work is reached)."""
import os

import pytest
import torch


def test_python_refusals():
    from ictc_o3 import layer_norm
    with pytest.raises(TypeError):
        layer_norm([1.0])
    with pytest.raises(ValueError, match="device"):
        layer_norm(torch.zeros(2, 4))


def test_native_refusals():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    size = nat.lib().ictc_layer_norm_workspace_bytes
    assert size(0, 100, 64) > 0 and size(1, 0, 16384) > 0
    assert size(3, 100, 64) == -1 and size(0, -1, 64) == -1 and size(0, 1, 0) == -1 and size(0, 1, 16385) == -1

    def fwd(dtype=0, ldx=64, rows=2, width=64, eps=1e-5, x=16):
        nat.call("ictc_layer_norm_fwd", dtype, x, ldx, rows, width, None, None, eps, x, None, None, None)

    for bad in (dict(dtype=5), dict(rows=-1), dict(width=0), dict(width=16385), dict(ldx=63), dict(eps=-1.0),
                dict(eps=float("nan")), dict(x=None)):
        with pytest.raises(ValueError):
            fwd(**bad)
    fwd(rows=0, x=None)
    with pytest.raises(ValueError, match="workspace"):
        nat.call("ictc_layer_norm_bwd", 0, 16, 64, 16, 64, 2, 64, None, 16, 16, None, 16, None, 16, 8, None)
    with pytest.raises(ValueError, match="workspace"):
        nat.call("ictc_layer_norm_bwd2", 0, 16, 64, 16, 64, 16, 64, None, None, 2, 64, None, 16, 16, None, None, 16,
                 None, 0, None)
