"""Traces of the dense layers' operators and of their backward passes are refused on the GPU too, and what is no trace
(a compiled function's graph break, a counting mode, recomputation) still runs."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


def _layers(device):
    from ictc_o3 import expert_linear, expert_order, layer_norm
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 16, generator=g).to(device).requires_grad_()
    w, W = torch.randn(16, generator=g).to(device), torch.randn(2, 24, 16, generator=g).to(device)
    order = expert_order(torch.randint(0, 2, (40,), generator=g).to(device), 2)
    return x, lambda t: layer_norm(t, w), lambda t: expert_linear(t, W, order)


def test_traces_are_refused(device):
    x, *layers = _layers(device)
    for layer in layers:
        for trace in (lambda: torch.jit.trace(layer, x, check_trace=False), lambda: make_fx(layer)(x)):
            with pytest.raises(ValueError, match="trac"):
                trace()
        y = layer(x)
        with pytest.raises(ValueError, match="trac"):
            make_fx(lambda g: torch.autograd.grad(y, x, g))(torch.ones_like(y))
        (first,) = torch.autograd.grad(layer(x), x, torch.ones_like(y), create_graph=True)
        if first.requires_grad:
            with pytest.raises(ValueError, match="trac"):
                make_fx(lambda v: torch.autograd.grad(first, x, v))(torch.ones_like(x))
        assert torch.equal(layer(x), y)


def test_what_is_no_trace_runs(device):
    from torch.utils.checkpoint import checkpoint
    from torch.utils.flop_counter import FlopCounterMode
    x, *layers = _layers(device)
    for layer in layers:
        y = layer(x)
        (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(torch.compile(lambda t: layer(t) + 0, backend="eager")(x), y)
        with FlopCounterMode(display=False):
            assert torch.equal(layer(x), y)
        again = checkpoint(layer, x, use_reentrant=False)
        assert torch.equal(again, y) and torch.equal(torch.autograd.grad(again, x, torch.ones_like(y))[0], gx)
