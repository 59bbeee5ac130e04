"""Refusals of the 8-bit activations' entry points (no GPU work is reached)."""
import os

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


def test_refusals():
    from ictc_o3 import _native as nat
    from ictc_o3 import decode_activations, encode_activations
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    with pytest.raises(TypeError):
        encode_activations([1.0])
    for call in (lambda: encode_activations(torch.zeros(2, 4)),
                 lambda: decode_activations(torch.zeros(2, 4, dtype=torch.int8), torch.zeros(2, 1))):
        with pytest.raises(ValueError, match="device"):
            call()
    for call in (lambda x: encode_activations(x), lambda x: decode_activations(x, x)):
        with pytest.raises(ValueError, match="trac"):
            make_fx(call)(torch.ones(2, 4))

    def encode(dtype=0, x=16, ldx=8, rows=2, width=8, codes=16, scales=16):
        nat.call("ictc_codes_encode", dtype, x, ldx, rows, width, codes, scales, None)

    def decode(dtype=0, codes=16, scales=16, rows=2, width=8, out=16):
        nat.call("ictc_codes_decode", dtype, codes, scales, rows, width, out, None)

    for bad in (dict(dtype=3), dict(x=None), dict(ldx=7), dict(rows=-1), dict(width=0), dict(codes=None),
                dict(scales=None)):
        with pytest.raises(ValueError):
            encode(**bad)
    for bad in (dict(dtype=-1), dict(codes=None), dict(scales=None), dict(rows=-1), dict(width=0), dict(out=None)):
        with pytest.raises(ValueError):
            decode(**bad)
    encode(rows=0, x=None, codes=None, scales=None)
    decode(rows=0, codes=None, scales=None, out=None)


def test_outer_refusals():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    takes = nat.lib().ictc_expert_outer_takes_codes
    assert takes(0, 32, 64, 10, 64, 32) and takes(1, 16, 8, 10, 8, 8)
    for bad in ((5, 32, 64, 10, 64, 32), (0, 8, 64, 10, 64, 32), (0, 32, 63, 10, 64, 32), (0, 32, 64, 0, 64, 32),
                (0, 32, 64, 10, 62, 32), (0, 32, 64, 10, 64, 30), (1, 32, 64, 10, 4, 8), (0, 32, 64, 10, 0, 32)):
        assert not takes(*bad), bad

    def outer(dtype=0, grad=16, ldg=8, codes=16, scales=16, rows=4, inputs=8, outputs=8, perm=16, off=16, out=16):
        nat.call("ictc_expert_outer_codes", dtype, grad, ldg, codes, scales, rows, inputs, outputs, 2, perm, off, out, None,
                 16, 1 << 30, None)

    for bad in (dict(dtype=3), dict(grad=None), dict(grad=20), dict(ldg=4), dict(ldg=9), dict(codes=None), dict(scales=None),
                dict(rows=0), dict(inputs=6), dict(outputs=6), dict(perm=None), dict(off=None), dict(out=None)):
        with pytest.raises(ValueError):
            outer(**bad)
