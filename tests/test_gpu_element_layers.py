"""The example that fits a potential with per-element layers: forces against differences of its energy, the gradient
of the force loss against differences of it, and both kinds of optimizer state bring the loss down."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _setup(device):
    import fit_element_layers as ex
    from ictc_o3 import expert_order
    data = ex.systems(1, 2, 3, device)
    model = ex.ElementPotential(seed=2, device=device)
    order = expert_order(data["element"], ex.ELEMENTS)

    def energy(pos):
        return model(pos, data["element"], order, data["src"], data["dst"], data["shift"]).double().sum()
    return data, model, energy


def test_forces_against_differences(device):
    """Central differences at 2^-6 A: truncation h^2 f'''/6 and rounding 2^-23 |E| / h are each below 1e-3 of the
    largest slope here; the bound is 1e-2 of the force norm times the step's."""
    data, _, energy = _setup(device)
    pos = data["pos"].clone().requires_grad_()
    (grad,) = torch.autograd.grad(energy(pos), pos)
    h = 2.0 ** -6
    for seed in range(3):
        d = torch.randn(pos.shape, generator=torch.Generator().manual_seed(seed)).to(device)
        d = d / d.norm()
        with torch.no_grad():
            diff = (energy(data["pos"] + h * d) - energy(data["pos"] - h * d)) / (2 * h)
        slope = (grad.double() * d.double()).sum()
        assert (diff - slope).abs() < 1e-2 * grad.double().norm()


def test_force_loss_gradient_against_differences(device):
    """The gradient of sum F^2 by every parameter at once, along random directions of relative length 2^-7."""
    data, model, energy = _setup(device)
    params = [p for p in model.parameters() if p.requires_grad]

    def loss(create):
        pos = data["pos"].clone().requires_grad_()
        (g,) = torch.autograd.grad(energy(pos), pos, create_graph=create)
        return g.square().sum().double()

    grads = torch.autograd.grad(loss(True), params, allow_unused=True)
    g = torch.Generator().manual_seed(5)
    start = [p.detach().clone() for p in params]
    step = [torch.randn(p.shape, generator=g).to(device) * p.detach().abs().mean() * 2.0 ** -7 for p in params]
    out = []
    for sign in (1, -1):
        with torch.no_grad():
            for p, s, d in zip(params, start, step):
                p.copy_(s + sign * d)
        out.append(loss(False))
    slope = sum((a.double() * d.double()).sum() for a, d in zip(grads, step) if a is not None)
    size = sum((a.double().square() * d.double().square()).sum() for a, d in zip(grads, step) if a is not None).sqrt()
    assert ((out[0] - out[1]) / 2 - slope).abs() < 2e-2 * torch.maximum(slope.abs(), size)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_brings_the_loss_down(device, bits):
    import fit_element_layers as ex
    _, history = ex.train(steps=120, cells=2, n=2, state_bits=bits, device=device)
    assert torch.isfinite(history).all()
    assert history[-10:, 1].mean() < 0.3 * history[:5, 1].mean()
