"""Layer norm against its formula in float64: output, gradients, gradients of the gradients, differences, refusals.

Bounds (max-norm, relative to the largest reference value), from the arithmetic: a row sum of w elements in at most
32 running terms per lane and ten tree levels is off by at most 42 units of 2^-24 relative to the sum of magnitudes,
and an output takes under ten more roundings, so FP32 results stay within 64 units of 2^-24 = 3.9e-6 where values and
statistics are of one size; the bound is 1e-5.  Parameter gradients add up to rows/16,384 + 100 further terms.
bfloat16 and float16 results are rounded once more: 2^-9 and 2^-11, the bounds are twice that.
"""
import pytest
import torch

from helpers import rel_err

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
EPS = 1e-5


def _formula(x, w, b, eps=EPS):
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    return y if b is None else y + b


def _inputs(rows, width, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + 0.3).to(dtype)
    w = (1 + 0.3 * torch.randn(width, generator=g)).to(dtype)
    b = (0.3 * torch.randn(width, generator=g)).to(dtype)
    gy, v = (torch.randn(rows, width, generator=g).to(dtype) for _ in range(2))
    return tuple(t.to(device) for t in (x, w, b, gy, v))


def _double(*ts):
    return tuple(None if t is None else t.detach().double().requires_grad_() for t in ts)


def _check(got, ref, dtype, names):
    for a, r, name in zip(got, ref, names):
        assert a.dtype == dtype and torch.isfinite(a).all(), name
        assert rel_err(a, r) < TOL[dtype], (name, rel_err(a, r))


# widths on both sides of every lane count, rows on both sides of a block's
WIDTHS = [1, 2, 7, 16, 63, 64, 65, 128, 129, 200, 256, 300, 512, 513, 1000, 1024, 2048, 2176, 4096, 5001, 8192, 16384]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", WIDTHS)
def test_output_and_gradients(device, width, dtype):
    from ictc_o3 import layer_norm
    for rows in (1, 37):
        x, w, b, gy, _ = _inputs(rows, width, dtype, width + rows, device)
        for t in (x, w, b):
            t.requires_grad_()
        y = layer_norm(x, w, b, eps=EPS)
        got = torch.autograd.grad(y, (x, w, b), gy)
        X, W, B = _double(x, w, b)
        Y = _formula(X, W, B)
        ref = torch.autograd.grad(Y, (X, W, B), gy.double())
        if width == 1:   # x equals its mean: y is the bias; no gradient reaches x or the weight
            assert torch.equal(y, b.detach().expand(rows, 1)) and got[0].abs().max() == 0 and got[1].abs().max() == 0
            assert rel_err(got[2], ref[2]) < TOL[dtype]
            continue
        if width == 2:   # dx cancels to eps / var of its terms, so FP32 keeps no relative accuracy of it
            _check((y, got[2]), (Y, ref[2]), dtype, ("y", "db"))
            continue
        _check((y, *got), (Y, *ref), dtype, ("y", "dx", "dw", "db"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [16, 64, 128, 200, 256, 512, 777, 2048, 2176, 8192, 9000])
def test_gradients_of_the_gradients(device, width, dtype):
    from ictc_o3 import layer_norm
    x, w, b, gy, v = _inputs(41, width, dtype, width, device)
    vw, vb = _inputs(2, width, dtype, width + 1, device)[1:3]
    for t in (x, w, b, gy):
        t.requires_grad_()
    first = torch.autograd.grad(layer_norm(x, w, b, eps=EPS), (x, w, b), gy, create_graph=True)
    X, W, B, G = _double(x, w, b, gy)
    First = torch.autograd.grad(_formula(X, W, B), (X, W, B), G, create_graph=True)
    for outs, cots in (((0,), (v,)), ((0, 1, 2), (v, vw, vb)), ((1,), (vw,)), ((1, 2), (vw, vb))):
        got = torch.autograd.grad([first[i] for i in outs], (x, gy), cots, retain_graph=True)
        ref = torch.autograd.grad([First[i] for i in outs], (X, G), [c.double() for c in cots], retain_graph=True)
        _check(got, ref, dtype, ("dx", "dg"))
    (got,) = torch.autograd.grad(first[0], w, v, retain_graph=True)
    (ref,) = torch.autograd.grad(First[0], W, v.double(), retain_graph=True)
    _check((got,), (ref,), dtype, ("dw",))


@pytest.mark.parametrize("rows,width", [(70001, 64), (4099, 1000)])
def test_many_rows(device, rows, width):
    from ictc_o3 import layer_norm
    x, w, b, gy, _ = _inputs(rows, width, torch.float32, 5, device)
    for t in (x, w, b):
        t.requires_grad_()
    y = layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), gy)
    again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), gy)
    assert all(torch.equal(i, j) for i, j in zip(got, again))       # a fixed order of every sum
    X, W, B = _double(x, w, b)
    Y = _formula(X, W, B)
    _check((y, *got), (Y, *torch.autograd.grad(Y, (X, W, B), gy.double())), torch.float32, ("y", "dx", "dw", "db"))


def test_absent_parameters_and_partial_gradients(device):
    from ictc_o3 import layer_norm
    x, w, b, gy, v = _inputs(19, 96, torch.float32, 3, device)
    for use_w, use_b in ((False, False), (True, False), (False, True)):
        ww, bb = w if use_w else None, b if use_b else None
        xr = x.clone().requires_grad_()
        y = layer_norm(xr, ww, bb)
        (gx,) = torch.autograd.grad(y, xr, gy, create_graph=True)
        (gxx,) = torch.autograd.grad(gx, xr, v)
        X, W, B = _double(x, ww, bb)
        Y = _formula(X, W, B)
        (GX,) = torch.autograd.grad(Y, X, gy.double(), create_graph=True)
        _check((y, gx, gxx), (Y, GX, torch.autograd.grad(GX, X, v.double())[0]), torch.float32, ("y", "dx", "dxx"))
    wr = w.clone().requires_grad_()
    (gw,) = torch.autograd.grad(layer_norm(x, wr, b), wr, gy)
    X, W, B = _double(x, w, b)
    _check((gw,), torch.autograd.grad(_formula(X, W, B), W, gy.double()), torch.float32, ("dw",))


def test_against_differences(device):
    """Central differences of the kernel's own output at step h: the truncation h^2 f'''/6 and the rounding
    2^-23 sqrt(terms) / h are both under 1e-3 of the gradient's norm at h = 2^-6; the bound is 1e-2."""
    from ictc_o3 import layer_norm
    x, w, b, gy, d = _inputs(5, 40, torch.float32, 9, device)
    h = 2.0 ** -6
    args = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*args), args, gy)
    for i in range(3):
        step = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(device)
        out = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(args)]
            out.append((layer_norm(*moved).double() * gy.double()).sum())
        diff = (out[0] - out[1]) / (2 * h)
        slope = (grads[i].double() * step.double()).sum()
        assert (diff - slope).abs() < 1e-2 * grads[i].double().norm() * step.double().norm()


def test_strides_and_leading_axes(device):
    from ictc_o3 import layer_norm
    x, w, b, gy, _ = _inputs(24, 70, torch.bfloat16, 4, device)
    plain = layer_norm(x, w, b)
    assert torch.equal(layer_norm(x.view(4, 6, 70), w, b), plain.view(4, 6, 70))
    wide = torch.zeros(24, 101, dtype=torch.bfloat16, device=device)
    wide[:, 3:73] = x                                        # rows at an odd pitch and an odd offset
    assert torch.equal(layer_norm(wide[:, 3:73], w, b), plain)
    assert torch.equal(layer_norm(x.t().contiguous().t(), w, b), plain)          # column-major
    assert torch.equal(layer_norm(x[:1].expand(24, 70), w, b), plain[:1].expand(24, 70))   # row pitch zero
    assert torch.equal(layer_norm(x[::2], w, b), plain[::2])
    assert torch.equal(layer_norm(x[3], w, b), plain[3])


def test_no_rows(device):
    from ictc_o3 import layer_norm
    x = torch.empty(0, 64, device=device, requires_grad=True)
    w, b = (torch.ones(64, device=device, requires_grad=True) for _ in range(2))
    y = layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y), create_graph=True)
    assert y.shape == (0, 64) and gx.shape == (0, 64)
    assert gw.abs().max() == 0 and gb.abs().max() == 0
    (ggw,) = torch.autograd.grad(gx, w, torch.empty_like(gx))
    assert ggw.abs().max() == 0


def test_rows_far_from_zero_and_rows_of_one_value(device):
    """A mean 4,096 times the spread costs 12 of FP32's 24 bits of x itself; the mean is removed before squares are
    added, so no more is lost: the inputs are exact multiples of 2^-11, and the bound stays 64 units of 2^-24 of
    the mean over the spread, 1.6e-2.  A row of one value has no spread: y is the bias, exactly."""
    from ictc_o3 import layer_norm
    g = torch.Generator().manual_seed(1)
    x = (4096 + torch.round(torch.randn(9, 512, generator=g) * 1024) / 1024).to(device)
    assert rel_err(layer_norm(x), _formula(x.double(), None, None)) < 1.6e-2
    b = torch.randn(512, generator=g).to(device)
    assert torch.equal(layer_norm(torch.full((3, 512), 2.5, device=device), None, b), b.expand(3, 512))


def test_nan_and_infinity_stay_in_their_rows(device):
    from ictc_o3 import layer_norm
    x, w, b, gy, _ = _inputs(33, 100, torch.float32, 2, device)
    clean = layer_norm(x, w, b)
    x[4, 17], x[20, 99] = float("nan"), float("inf")
    y = layer_norm(x, w, b)
    bad = torch.zeros(33, dtype=torch.bool, device=device)
    bad[[4, 20]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


def test_third_derivative_raises(device):
    from ictc_o3 import layer_norm
    x = torch.randn(4, 32, device=device, requires_grad=True)
    (g1,) = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    (g2,) = torch.autograd.grad(g1.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g2.sum(), x)


def test_graph_replays_and_side_streams(device):
    from ictc_o3 import layer_norm
    x, w, b, gy, _ = _inputs(300, 64, torch.float32, 8, device)
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        y = layer_norm(x, w, b)
        return (y, *torch.autograd.grad(y, (x, w, b), gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.add_(0.25)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) for i, j in zip(held, eager)), k


def test_offsets_past_32_bits(device):
    """More than 2^31 elements: the first and last rows and their gradients alone."""
    from ictc_o3 import layer_norm
    N, C = 34000000, 64
    g = torch.Generator(device).manual_seed(1)
    x = torch.randn(N, C, device=device, generator=g).requires_grad_()
    w, b = (torch.randn(C, device=device, generator=g).requires_grad_() for _ in range(2))
    y = layer_norm(x, w, b)
    ends = torch.cat([torch.arange(0, 200, device=device), torch.arange(N - 200, N, device=device)])
    gy = torch.zeros(N, C, device=device)
    gy[ends] = torch.randn(400, C, device=device, generator=g)
    got = torch.autograd.grad(y, (x, w, b), gy)
    few = [t.detach().double().requires_grad_() for t in (x[ends], w, b)]
    Y = torch.nn.functional.layer_norm(few[0], (C,), few[1], few[2])
    ref = torch.autograd.grad(Y, few, gy[ends].double())
    for a, r in zip((y[ends], got[0][ends], got[1], got[2]), (Y, *ref)):
        assert rel_err(a, r) < TOL[torch.float32]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_without_a_graph(device, dtype):
    from ictc_o3 import layer_norm
    x, w, b, _, _ = _inputs(77, 130, dtype, 5, device)
    plain = layer_norm(x, w, b)
    kept = layer_norm(x, w.clone().requires_grad_(), b)
    with torch.no_grad():
        off = layer_norm(x.clone().requires_grad_(), w, b)
    with torch.inference_mode():
        inference = layer_norm(x, w, b)
    assert kept.requires_grad and not plain.requires_grad and not off.requires_grad
    assert all(torch.equal(t, kept) for t in (plain, off, inference))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(36011, 64), (36011, 120), (20011, 250), (9001, 500), (5003, 1000),
                                        (5003, 2000), (2531, 2176), (2531, 4096), (1201, 8192), (1201, 9000),
                                        (601, 16384)])
def test_rows_that_a_team_takes_in_turn(device, rows, width, dtype):
    """Rows enough that every team of every kernel has several, the last round part full: results, gradients and
    gradients of the gradients, the latter two with their sums over rows."""
    from ictc_o3 import layer_norm
    x, w, b, gy, v = _inputs(rows, width, dtype, 5, device)
    vw, vb = _inputs(2, width, dtype, 6, device)[1:3]
    for t in (x, w, b, gy):
        t.requires_grad_()
    X, W, B, G = _double(x, w, b, gy)
    y, Y = layer_norm(x, w, b, eps=EPS), _formula(X, W, B)
    first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
    First = torch.autograd.grad(Y, (X, W, B), G, create_graph=True)
    _check((y, *first), (Y, *First), dtype, ("y", "dx", "dw", "db"))
    second = torch.autograd.grad(first, (x, gy), (v, vw, vb), retain_graph=True)
    _check(second, torch.autograd.grad(First, (X, G), (v.double(), vw.double(), vb.double()), retain_graph=True), dtype,
           ("dx'", "dg'"))
    second = torch.autograd.grad(first[0], (x, w, gy), v)
    _check(second, torch.autograd.grad(First[0], (X, W, G), v.double()), dtype, ("dx'", "dw'", "dg'"))


@pytest.mark.parametrize("width", [16, 64, 128, 200, 256, 512, 777, 2048, 2176, 8192, 9000])
def test_gradients_of_the_gradients_in_half(device, width):
    from ictc_o3 import layer_norm
    dtype = torch.float16
    x, w, b, gy, v = _inputs(41, width, dtype, width, device)
    vw, vb = _inputs(2, width, dtype, width + 1, device)[1:3]
    for t in (x, w, b, gy):
        t.requires_grad_()
    first = torch.autograd.grad(layer_norm(x, w, b, eps=EPS), (x, w, b), gy, create_graph=True)
    X, W, B, G = _double(x, w, b, gy)
    First = torch.autograd.grad(_formula(X, W, B), (X, W, B), G, create_graph=True)
    for outs, cots in (((0,), (v,)), ((0, 1, 2), (v, vw, vb)), ((1,), (vw,)), ((1, 2), (vw, vb))):
        got = torch.autograd.grad([first[i] for i in outs], (x, gy), cots, retain_graph=True)
        ref = torch.autograd.grad([First[i] for i in outs], (X, G), [c.double() for c in cots], retain_graph=True)
        _check(got, ref, dtype, ("dx", "dg"))
    (got,) = torch.autograd.grad(first[0], w, v, retain_graph=True)
    (ref,) = torch.autograd.grad(First[0], W, v.double(), retain_graph=True)
    _check((got,), (ref,), dtype, ("dw",))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [40, 100, 250, 500, 1000, 2000, 2176, 8192, 9000])
def test_rows_whose_squares_leave_the_range(device, width, dtype):
    """Finite rows spread over up to 2^110, whose variance FP32 does not hold, beside ordinary ones: a power of two
    changes no rounding, so the bounds are the ordinary ones, row by row."""
    from ictc_o3 import layer_norm
    x, w, b, gy, _ = _inputs(40, width, dtype, 3, device)
    size = torch.exp2(torch.tensor([0.0, 62.0, 66.0, 90.0, 110.0], device=device)).repeat(8)[:, None]
    x = (x.float() * size).to(dtype).requires_grad_()
    y = layer_norm(x, w, b)
    (gx,) = torch.autograd.grad(y, x, gy)
    X, W, B = _double(x, w, b)
    Y = _formula(X, W, B)
    (GX,) = torch.autograd.grad(Y, X, gy.double())
    _check((y,), (Y,), dtype, ("y",))
    assert rel_err(gx.double() * size, GX * size) < TOL[dtype]
