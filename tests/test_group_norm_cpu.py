"""The written-out derivatives of the group norm against autograd, and refusals of its entry points (no GPU work)."""
import os

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from group_norm_formulas import Derivatives, definition


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("shape,groups", [((3, 12), 3), ((2, 5, 8), 2), ((2, 3, 2, 6), 6), ((4, 7), 1)])
def test_derivatives_against_autograd(shape, groups, activation):
    g = torch.Generator().manual_seed(1)
    x, gy, v = (torch.randn(shape, generator=g, dtype=torch.float64).requires_grad_() for _ in range(3))
    w, b, vw, vb = (torch.randn(shape[-1], generator=g, dtype=torch.float64).requires_grad_() for _ in range(4))
    first = torch.autograd.grad(definition(x, groups, w, b, 1e-2, activation), (x, w, b), gy, create_graph=True)
    d = Derivatives(x.detach(), groups, w.detach(), b.detach(), 1e-2, activation, gy.detach())
    for got, ref in zip(d.first()[0], first):
        assert (got - ref).abs().max() < 1e-10
    second = torch.autograd.grad(first, (x, gy, w, b), (v, vw, vb), allow_unused=True)
    for got, ref in zip(d.second(v.detach(), vw.detach(), vb.detach())[0], second):
        assert (got - (0 if ref is None else ref)).abs().max() < 1e-10


def test_python_refusals():
    from ictc_o3 import _native as nat
    from ictc_o3 import group_norm
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    with pytest.raises(TypeError):
        group_norm([1.0], 1)
    with pytest.raises(ValueError, match="device"):
        group_norm(torch.zeros(2, 4), 1)
    with pytest.raises(ValueError, match="trac"):
        make_fx(lambda x: group_norm(x, 2))(torch.ones(2, 4))
    with pytest.raises(ValueError, match="trac"):
        torch.jit.trace(lambda x: group_norm(x, 2), torch.ones(2, 4), check_trace=False)


def test_native_refusals():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    size = nat.lib().ictc_group_norm_workspace_bytes
    assert size(0, 0, 100, 1, 64, 8) == 0 and size(0, 1, 100, 1, 64, 8) > 0 and size(1, 2, 0, 5, 64, 8) > 0
    assert size(0, 0, 1, 100000, 64, 8) > 0
    for bad in ((3, 0, 1, 1, 4, 1), (0, 3, 1, 1, 4, 1), (0, -1, 1, 1, 4, 1), (0, 0, -1, 1, 4, 1), (0, 0, 1, -1, 4, 1),
                (0, 0, 1, 1, 0, 1), (0, 0, 1, 1, 65537, 1), (0, 0, 1, 1, 4, 3), (0, 0, 1, 1, 4, 0),
                (0, 0, 2 ** 39, 2 ** 39, 4, 1)):
        assert size(*bad) == -1, bad

    def fwd(dtype=0, x=16, samples=2, positions=3, channels=8, groups=2, eps=1e-5, act=0, y=16, mean=None, rstd=None,
            codes=None, scales=None, ws=None, bytes=0):
        nat.call("ictc_group_norm_fwd", dtype, x, samples, positions, channels, groups, None, None, eps, act, y, mean,
                 rstd, codes, scales, ws, bytes, None)

    for bad in (dict(dtype=4), dict(x=None), dict(samples=-1), dict(positions=-1), dict(channels=0), dict(groups=3),
                dict(eps=-1.0), dict(eps=float("nan")), dict(act=2), dict(y=None), dict(mean=16),
                dict(codes=16), dict(scales=16),
                dict(samples=1, positions=100000)):
        with pytest.raises(ValueError):
            fwd(**bad)
    fwd(samples=0, x=None, y=None)
    fwd(positions=0, x=None, y=None)

    def bwd(name="ictc_group_norm_bwd", x=16, codes=None, scales=None, grad=16, v=(), samples=2, act=0, mean=16, rstd=16,
            out=(16, 16, 16), ws=16, bytes=1 << 20):
        nat.call(name, 0, x, codes, scales, grad, *v, samples, 3, 8, 2, None, None, act, mean, rstd, *out, ws, bytes, None)

    second = dict(name="ictc_group_norm_bwd2", v=(16, None, None), out=(16, 16, 16, 16))
    for more in ({}, second):
        for bad in (dict(x=None), dict(codes=16), dict(x=None, codes=16), dict(grad=None), dict(samples=-1), dict(act=-1),
                    dict(mean=None), dict(rstd=None), dict(ws=None), dict(ws=20), dict(bytes=8)):
            with pytest.raises(ValueError):
                bwd(**{**more, **bad})
    with pytest.raises(ValueError):
        bwd(**{**second, "v": (None, None, None)})
    bwd(out=(None, None, None))


def test_native_refusals_of_the_means_rest():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    keeps = nat.lib().ictc_group_norm_keeps_rest
    assert keeps(0, 3, 300, 64, 8) and keeps(0, 1, 100000, 64, 8) and not keeps(0, 100, 1, 64, 8)
    for none in ((1, 3, 300, 64, 8), (2, 3, 300, 64, 8), (0, 0, 300, 64, 8), (0, 3, 0, 64, 8), (0, 3, 300, 64, 7), (4, 3, 300, 64, 8)):
        assert not keeps(*none), none

    def fwd(mean=16, rest=16, rstd=16, x=16, samples=2):
        nat.call("ictc_group_norm_fwd_rest", 0, x, samples, 3, 8, 2, None, None, 1e-5, 0, 16, mean, rest, rstd, None, None,
                 None, 0, None)

    for bad in (dict(mean=None), dict(mean=None, rstd=None), dict(rstd=None), dict(x=None), dict(samples=-1)):
        with pytest.raises(ValueError):
            fwd(**bad)
    fwd(samples=0)
    for name, v, out in (("ictc_group_norm_bwd_rest", (), (16, 16, 16)),
                         ("ictc_group_norm_bwd2_rest", (16, None, None), (16, 16, 16, 16))):
        for mean, rstd, ws in ((None, 16, 16), (16, None, 16), (16, 16, None)):
            with pytest.raises(ValueError):
                nat.call(name, 0, 16, None, None, 16, *v, 2, 3, 8, 2, None, None, 0, mean, 16, rstd, *out, ws, 1 << 20, None)
