"""Fits a small interatomic potential whose atomic layers are chosen by element, on energies and forces.

    python examples/fit_element_layers.py [--steps 300] [--state-bits 8] [--cells 4]

Each atom gathers its neighbours with the graph message (degree 0 and 1 harmonics, radial gates), the invariants of
the result go through layer norm, a linear of the atom's own element, SiLU and a second such linear to an atomic
energy, and forces are minus the gradient by the positions.  The loss on forces differentiates that gradient again, so
the norm and the element linears run forward, backward and through their second derivatives; AdamW updates all
parameters at once with the gradients' norm bounded.  The data are jittered FCC cells of four elements under a pair
potential with element-dependent strengths.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ictc-o3-hp-k100_amd")
if PKG not in sys.path:
    sys.path.insert(0, PKG)

from ictc_o3 import (AdamW, PackedGraphMessage, direction_harmonics, expert_linear, expert_order,  # noqa: E402
                     layer_norm, normalized_silu)
from ictc_o3.ops.activation import radial_embedding  # noqa: E402
from mace_ictc.hp import radius_graph_pbc  # noqa: E402

CUTOFF, ELEMENTS, DENSITY = 4.5, 4, 0.1


def systems(cells, n, seed, device):
    """`cells` jittered FCC boxes of 4 n^3 atoms as one batch, with energies and forces of the pair potential."""
    g = torch.Generator().manual_seed(seed)
    a = (4.0 / DENSITY) ** (1.0 / 3.0)
    base = torch.tensor([[0, 0, 0], [0.5, 0.5, 0], [0.5, 0, 0.5], [0, 0.5, 0.5]])
    grid = torch.stack(torch.meshgrid(*[torch.arange(float(n))] * 3, indexing="ij"), -1).reshape(-1, 1, 3)
    box = torch.eye(3) * a * n
    pos, src, dst, shift, atoms = [], [], [], [], 0
    for _ in range(cells):
        p = ((grid + base).reshape(-1, 3) * a + 0.3 * torch.randn(4 * n ** 3, 3, generator=g)).to(device)
        s, d, sh = radius_graph_pbc(p, box.to(device), CUTOFF)
        pos.append(p)
        src.append(s + atoms)
        dst.append(d + atoms)
        shift.append(sh.float() @ box.to(device))
        atoms += p.shape[0]
    data = dict(pos=torch.cat(pos), src=torch.cat(src), dst=torch.cat(dst), shift=torch.cat(shift),
                element=torch.randint(0, ELEMENTS, (atoms,), generator=g).to(device))
    strength = torch.randn(ELEMENTS, ELEMENTS, generator=torch.Generator().manual_seed(1)).to(device)
    strength = strength + strength.t()
    p = data["pos"].double().requires_grad_()
    r = (p[data["dst"]] - p[data["src"]] + data["shift"].double()).norm(dim=1)
    pair = strength[data["element"][data["src"]], data["element"][data["dst"]]].double()
    energy = torch.zeros(atoms, dtype=torch.float64, device=device).index_add(
        0, data["dst"], pair * torch.exp(-(r / 1.8) ** 2) * torch.cos(math.pi * r / (2 * CUTOFF)))
    data["forces"] = -torch.autograd.grad(energy.sum(), p)[0].float()
    data["energy"] = energy.detach().float().view(cells, -1).sum(1)
    return data


class ElementPotential(torch.nn.Module):
    def __init__(self, channels=32, hidden=64, seed=0, device="cuda"):
        super().__init__()
        self.message = PackedGraphMessage.create(channels=channels, input_lmax=0, edge_lmax=1, output_lmax=1,
                                                 device=device)
        self.channels = channels
        g = torch.Generator().manual_seed(seed)

        def weight(*shape):
            return torch.nn.Parameter((torch.randn(*shape, generator=g) / math.sqrt(shape[-1])).to(device))

        def norm(width):
            return torch.nn.ParameterList([torch.nn.Parameter(torch.ones(width, device=device)),
                                           torch.nn.Parameter(torch.zeros(width, device=device))])

        self.embedding = weight(ELEMENTS, channels)
        self.radial_1, self.radial_norm = weight(hidden, 8), norm(hidden)
        self.radial_2 = weight(self.message.gate_width, hidden)
        self.node_norm = norm(2 * channels)
        self.weight_1, self.bias_1 = weight(ELEMENTS, hidden, 2 * channels), weight(ELEMENTS, hidden)
        self.weight_2, self.bias_2 = weight(ELEMENTS, 1, hidden), weight(ELEMENTS, 1)

    def forward(self, pos, element, order, src, dst, shift):
        """Atomic energies [N]; `order` is expert_order(element, ELEMENTS), shared by every step of a batch."""
        vec = pos[dst] - pos[src] + shift
        r = vec.norm(dim=1)
        harmonics = torch.cat(direction_harmonics(vec / r[:, None], 1), 1)
        radial = normalized_silu(layer_norm(radial_embedding(r, CUTOFF) @ self.radial_1.t(), *self.radial_norm))
        # (the norm undoes the basis' decay towards the cutoff: the gates get it back)
        gates = (radial @ self.radial_2.t()) * (0.5 + 0.5 * torch.cos(math.pi * r / CUTOFF))[:, None]
        m = self.message(self.embedding[element], harmonics, gates, src, dst)
        scalars, vectors = m[:, :self.channels], m[:, self.channels:].reshape(-1, 3, self.channels)
        x = layer_norm(torch.cat([scalars, (vectors * vectors).sum(1)], 1), *self.node_norm)
        x = normalized_silu(expert_linear(x, self.weight_1, order, self.bias_1))
        return expert_linear(x, self.weight_2, order, self.bias_2).squeeze(1)


def train(steps=300, cells=4, n=3, state_bits=32, lr=4e-3, seed=0, device="cuda", log=None):
    """(model, [(energy loss, force loss, gradient norm) of each step])."""
    torch.manual_seed(seed)
    data = systems(cells, n, seed, device)
    model = ElementPotential(seed=seed, device=device)
    opt = AdamW([p for p in model.parameters() if p.requires_grad], lr=lr, weight_decay=1e-4, max_norm=10.0,
                state_bits=state_bits)
    order = expert_order(data["element"], ELEMENTS)
    atoms = data["pos"].shape[0] // cells
    history = []
    # A system as small as these is bound by its host: backward passes in this thread, not handed over to the engine's
    # (3.6 to 4.5 ms a step with it, 2.8 to 3.0 without).
    with torch.autograd.set_multithreading_enabled(False):
        for k in range(steps):
            pos = data["pos"].requires_grad_()
            energy = model(pos, data["element"], order, data["src"], data["dst"], data["shift"])
            forces = -torch.autograd.grad(energy.sum(), pos, create_graph=True)[0]
            e_loss = ((energy.view(cells, -1).sum(1) - data["energy"]) / atoms).square().mean()
            f_loss = (forces - data["forces"]).square().mean()
            opt.zero_grad()
            (e_loss + 10 * f_loss).backward(inputs=[p for p in model.parameters() if p.requires_grad])
            opt.step()
            history.append(torch.stack([e_loss.detach(), f_loss.detach(), opt.grad_norm]))
            if log and (k % 50 == 0 or k == steps - 1):
                e, f, norm = history[-1].tolist()
                log(f"step {k:4d}  energy loss {e:.5f} per atom^2  force loss {f:.5f}  gradient norm {norm:.3f}")
    return model, torch.stack(history).cpu()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--cells", type=int, default=4)
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    a = ap.parse_args()
    train(a.steps, a.cells, state_bits=a.state_bits, log=lambda text: print(text, flush=True))
