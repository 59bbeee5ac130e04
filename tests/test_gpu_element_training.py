"""The layers of an element network together, as a training step on energies and forces runs them: embedding, per-element
linears, group norm with SiLU, and another linear; the rows kept whole or in 8 bits.

Bounds.  An output of the step has passed six operators whose own results are within 4e-5 of their largest value at most
(the second derivative of the group norm), so the step's gradients are held to 3e-4 in the max-norm.  In 8 bits a value is
off by 1/254 of its block's largest at most, some 1.7 % of the root mean square of normal values, evenly spread, so about
1 % root mean square; three kept tensors add up to 3 % at most of a gradient's norm: the bound is 5 %.
"""
import pytest
import torch

from group_norm_formulas import definition
from helpers import rel_err

pytestmark = pytest.mark.gpu
ELEMENTS, WIDTH, HIDDEN, GROUPS = 6, 64, 128, 8


def _data(atoms, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    element = torch.randint(0, ELEMENTS, (atoms,), generator=g)
    if atoms > 3:
        element[atoms // 2] = -1                       # an atom of no element
    field = torch.randn(atoms, WIDTH, generator=g)
    shapes = dict(table=(ELEMENTS, WIDTH), w1=(ELEMENTS, HIDDEN, WIDTH), b1=(ELEMENTS, HIDDEN), gamma=(HIDDEN,), beta=(HIDDEN,),
                  w2=(ELEMENTS, 1, HIDDEN), b2=(ELEMENTS, 1))
    p = {name: torch.randn(shape, generator=g) / (shape[-1] ** 0.5 if name[0] == "w" else 3.0) for name, shape in shapes.items()}
    p["gamma"] = 1 + 0.2 * p["gamma"]
    return element.to(device), field.to(device), {name: t.to(device) for name, t in p.items()}


def _step(element, field, p, bits=None):
    """(energy, forces on the field, gradients of all parameters) of one training step."""
    from ictc_o3 import embedding, expert_linear, expert_order, group_norm
    p = {name: t.detach().requires_grad_() for name, t in p.items()}
    field = field.detach().requires_grad_()
    order = expert_order(element, ELEMENTS)
    x = embedding(p["table"], element, 2.0, order=order) * field
    x = expert_linear(x, p["w1"], order, p["b1"], save_bits=bits)
    x = group_norm(x, GROUPS, p["gamma"], p["beta"], activation="silu", save_bits=bits)
    energy = expert_linear(x, p["w2"], order, p["b2"], save_bits=bits).sum()
    (force,) = torch.autograd.grad(energy, field, create_graph=True)
    loss = 0.1 * energy.square() + force.square().sum()
    grads = torch.autograd.grad(loss, list(p.values()))
    return (energy.detach(), force.detach(), *grads)


def _reference(element, field, p):
    p = {name: t.double().requires_grad_() for name, t in p.items()}
    field = field.double().requires_grad_()
    valid = (element >= 0)[:, None].double()
    at = element.clamp(min=0)
    x = 2.0 * p["table"][at] * valid * field
    x = ((p["w1"][at] @ x[:, :, None]).squeeze(2) + p["b1"][at]) * valid
    x = definition(x, GROUPS, p["gamma"], p["beta"], 1e-5, "silu")
    energy = (((p["w2"][at] @ x[:, :, None]).squeeze(2) + p["b2"][at]) * valid).sum()
    (force,) = torch.autograd.grad(energy, field, create_graph=True)
    loss = 0.1 * energy.square() + force.square().sum()
    return (energy.detach(), force.detach(), *torch.autograd.grad(loss, list(p.values())))


@pytest.mark.parametrize("atoms", [1, 5, 300, 4001])
def test_step_against_float64(device, atoms):
    element, field, p = _data(atoms, device)
    for got, ref in zip(_step(element, field, p), _reference(element, field, p)):
        assert got.shape == ref.shape and rel_err(got, ref) < 3e-4


@pytest.mark.parametrize("atoms", [300, 4001])
def test_step_with_rows_in_8_bits(device, atoms):
    element, field, p = _data(atoms, device)
    whole, eight = _step(element, field, p), _step(element, field, p, 8)
    assert torch.equal(whole[0], eight[0])
    again = _step(element, field, p, 8)
    for a, b, c in zip(eight, whole, again):
        assert torch.equal(a, c)
        assert (a.double() - b.double()).norm() <= 0.05 * b.double().norm()


@pytest.mark.parametrize("bits", [None, 8])
def test_captured_and_replayed(device, bits):
    element, field, p = _data(700, device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(element, field, p, bits)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(element, field, p, bits)
    for k in range(3):
        field.mul_(-0.75).add_(0.1)
        element.copy_(element.roll(17))
        p["w1"].mul_(1.1)
        graph.replay()
        eager = _step(element, field, p, bits)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_two_streams_at_once(device):
    """Steps of different data on two streams, and two graphs replayed at once, give what they give alone."""
    inputs = [_data(2500, device, seed) for seed in (1, 2)]
    alone = [_step(*i, 8) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    for _ in range(3):
        out = []
        for i, stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                out.append(_step(*i, 8))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(out, alone) for a, b in zip(x, y))
    del out
    graphs, held = [], []
    for i in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(_step(*i, 8))
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(held, alone) for a, b in zip(x, y))


def test_traces_are_refused(device):
    from torch.fx.experimental.proxy_tensor import make_fx
    from ictc_o3 import embedding, group_norm
    element, field, p = _data(40, device)
    table = p["table"].requires_grad_()
    x = field.requires_grad_()
    for f, t in ((lambda t: embedding(t, element), table), (lambda t: group_norm(t, 8), x),
                 (lambda t: group_norm(t, 8, save_bits=8), x)):
        for trace in (lambda: torch.jit.trace(f, t, check_trace=False), lambda: make_fx(f)(t)):
            with pytest.raises(ValueError, match="trac"):
                trace()
        y = f(t)
        with pytest.raises(ValueError, match="trac"):
            make_fx(lambda g: torch.autograd.grad(y, t, g))(torch.ones_like(y))


def test_recomputed_and_in_threads(device):
    """Under torch's own checkpoint the layers run again and give the same gradients; so do calls of several threads."""
    import threading
    from torch.utils.checkpoint import checkpoint
    from ictc_o3 import group_norm
    x = torch.randn(200, 64, device=device, requires_grad=True)
    w = torch.randn(64, device=device, requires_grad=True)
    gy = torch.randn(200, 64, device=device)

    def layer(t):
        return group_norm(t, 8, w, activation="silu", save_bits=8)
    ref = torch.autograd.grad(layer(x), (x, w), gy)
    got = torch.autograd.grad(checkpoint(layer, x, use_reentrant=False), (x, w), gy)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                out = torch.autograd.grad(layer(x), (x, w), gy)
            torch.cuda.current_stream().synchronize()
            results[i] = out
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for out in results for a, b in zip(out, ref))


def test_example_with_group_norm(device):
    """The example's form with the embedding, group norm and 8 bits: it runs, and its forces are its energy's slopes (central
    differences at 2^-6 A, bounds as of its other form)."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import fit_element_layers as ex
    from ictc_o3 import expert_order
    for bits in (None, 8):
        _, history = ex.train(steps=3, cells=1, n=2, device=device, groups=8, save_bits=bits)
        assert torch.isfinite(history).all()
    data = ex.systems(1, 2, 3, device)
    model = ex.ElementPotential(seed=2, device=device, groups=8)
    order = expert_order(data["element"], ex.ELEMENTS)

    def energy(pos):
        return model(pos, data["element"], order, data["src"], data["dst"], data["shift"]).double().sum()
    pos = data["pos"].clone().requires_grad_()
    (grad,) = torch.autograd.grad(energy(pos), pos)
    h = 2.0 ** -6
    for seed in range(3):
        d = torch.randn(pos.shape, generator=torch.Generator().manual_seed(seed)).to(device)
        d = d / d.norm()
        with torch.no_grad():
            diff = (energy(data["pos"] + h * d) - energy(data["pos"] - h * d)) / (2 * h)
        assert (diff - (grad.double() * d.double()).sum()).abs() < 1e-2 * grad.double().norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [64, 130])
def test_operands_that_begin_anywhere(device, width, dtype):
    """Contiguous operands one element behind an aligned address: the results of aligned ones, bit by bit."""
    from ictc_o3 import decode_activations, embedding, encode_activations, group_norm
    generator = torch.Generator().manual_seed(width)

    def make(*size):
        return torch.randn(*size, generator=generator).to(dtype).to(device)

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=device)
        flat[1:] = t.detach().reshape(-1)
        return flat[1:].view(t.shape).requires_grad_(t.requires_grad)

    ids = torch.randint(-1, 12, (700,), generator=generator).to(device)

    def run(at):
        table, g = at(make_table).requires_grad_(), at(make_g)
        rows = embedding(table, at(ids), 0.75)
        out = [rows, *torch.autograd.grad(rows, table, g)]
        for x, gy, bits in ((make_x, make_g, None), (make_cells, make_cells_g, None), (make_x, make_g, 8)):
            x, w, b, gy, v = at(x).requires_grad_(), at(make_w).requires_grad_(), at(make_b).requires_grad_(), at(gy), at(gy)
            y = group_norm(x, 2, w, b, activation="silu", save_bits=bits)
            first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
            out += [y, *first, *torch.autograd.grad(first[0], (x, w), v)]
        codes, scales = encode_activations(at(make_x))
        return [*out, codes, scales, decode_activations(at(codes), at(scales), dtype=dtype)]

    make_table, make_g, make_x, make_w, make_b = make(12, width), make(700, width), make(700, width), make(width), make(width)
    make_cells, make_cells_g = make(3, 500, width), make(3, 500, width)
    for a, b in zip(run(lambda t: t.detach()), run(moved)):
        assert torch.equal(a, b)
