"""Group norm with an activation against its formulas in float64: output, gradients, gradients of the gradients, 8 bits.

Bounds.  Row results (max-norm, relative to the largest reference value): a group's sums are off by at most d units of
2^-24 of the sum of magnitudes, d the longest chain of additions: 32 in a lane of the rows' form, some hundred in a
thread of the others' (of alternating sign, so that a few tens are reached), ten levels of a tree; the activation adds
under ten, of which the exponential's argument has 1.5 |z|.  64 units are 3.9e-6; the bound is 1e-5, and four times that
for the second derivative, which has four such sums one behind another.  Sums over samples (dw, db): 600 units of 2^-24
of the sum of their terms' magnitudes, 512 in a thread and the rest in trees.  bfloat16 and float16 round once more by
half a step; the bounds are a step, 2^-8 and 2^-10.
"""
import pytest
import torch

from group_norm_formulas import Derivatives, definition
from helpers import rel_err

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
SECOND = {**TOL, torch.float32: 4e-5}
EPS = 1e-5

SHAPES = [  # samples, positions, channels, groups: one position
    (1, 1, 4, 1), (37, 1, 64, 8), (3, 1, 64, 64), (5, 1, 30, 5), (9, 1, 35, 5), (9, 1, 96, 4), (33, 1, 13, 1),
    (3, 1, 512, 1), (4, 1, 1024, 2), (3, 1, 1000, 1), (3, 1, 2048, 1), (5, 1, 600, 200), (1100, 1, 24, 3),
    (3, 1, 2176, 1), (5, 1, 8192, 2), (2, 1, 5001, 1), (0, 1, 16, 4),
    (3, 1, 8192, 1), (5, 1, 4096, 1), (4, 1, 6144, 2), (2, 1, 16384, 1), (4, 1, 999, 3), (7, 1, 77, 7), (3, 1, 1010, 1),
    (5, 1, 45, 5), (3, 1, 2001, 1), (6, 1, 18, 3), (4, 1, 33, 3),
    # a few positions
    (9, 5, 45, 5), (7, 3, 77, 7), (5, 4, 26, 2), (11, 9, 128, 8), (5, 16, 90, 3), (3, 25, 27, 3), (4, 7, 1022, 2),
    (7, 9, 64, 8), (3, 128, 16, 2), (5, 33, 30, 5), (6, 2, 7, 7), (4, 16, 64, 2), (2, 3, 256, 1), (50, 5, 36, 12),
    # blocks, one sample after another or many
    (3, 300, 64, 8), (2, 257, 330, 11), (40, 200, 48, 2), (700, 140, 40, 1), (3, 513, 5, 5), (2, 100, 900, 3),
    (1, 65, 2048, 8),
    (30, 70, 64, 64), (3, 400, 14, 7), (5, 300, 36, 12),
    # parts
    (1, 5000, 64, 8), (2, 4099, 30, 5), (1, 700, 2304, 1), (2, 3, 8000, 2), (1, 20011, 12, 4), (3, 1, 65536, 1),
    (2, 0, 8, 2)]


def _inputs(shape, dtype, device, seed=0):
    samples, positions, channels, _ = shape
    g = torch.Generator().manual_seed(seed + sum(shape))
    size = (samples, positions, channels) if positions != 1 else (samples, channels)
    x = (torch.randn(size, generator=g) * (0.5 + torch.rand(samples, *[1] * (len(size) - 1), generator=g)) + 0.3)
    w, b, vw, vb = (torch.randn(channels, generator=g) * 0.3 for _ in range(4))
    gy, v = (torch.randn(size, generator=g) for _ in range(2))
    return tuple(t.to(dtype).to(device) for t in (x, 1 + w, b, gy, v, vw, vb))


def _close(got, ref, tol, name):
    assert torch.isfinite(got).all(), name
    assert got.numel() == 0 or rel_err(got, ref) < tol, (name, rel_err(got, ref))


def _close_sum(got, ref, size, name):
    unit = torch.finfo(got.dtype).eps
    bound = 600 * 2.0 ** -24 * size + (unit if got.dtype != torch.float32 else 0) * ref.abs() + 1e-30
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    worst = ((got.double() - ref).abs() / bound).max()
    assert torch.isfinite(got).all() and worst <= 1, (name, float(worst))


def _few(shape):
    """Groups of so few elements that the input gradient cancels to eps / var of its terms: no relative accuracy."""
    return shape[1] * (shape[2] // shape[3]) <= 3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_output_and_gradients(device, shape, dtype):
    from ictc_o3 import group_norm
    x, w, b, gy, *_ = _inputs(shape, dtype, device)
    for t in (x, w, b):
        t.requires_grad_()
    for activation in (None, "silu"):
        y = group_norm(x, shape[3], w, b, eps=EPS, activation=activation)
        got = torch.autograd.grad(y, (x, w, b), gy)
        assert y.shape == x.shape and all(t.dtype == dtype for t in (y, *got))
        if x.numel():
            ref = definition(x.detach().double(), shape[3], w.detach().double(), b.detach().double(), EPS, activation)
            _close(y, ref, TOL[dtype], "y")
        else:
            assert all((t == 0).all() for t in got)
            continue
        (dx, dw, db), (sw, sb) = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, activation, gy).first()
        if not _few(shape):
            _close(got[0], dx, TOL[dtype], "dx")
            _close_sum(got[1], dw, sw, "dw")
        _close_sum(got[2], db, sb, "db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [s for s in SHAPES if not _few(s) and s[0]])
def test_gradients_of_the_gradients(device, shape, dtype):
    from ictc_o3 import group_norm
    x, w, b, gy, v, vw, vb = _inputs(shape, dtype, device)
    for t in (x, w, b, gy):
        t.requires_grad_()
    for activation in (None, "silu"):
        y = group_norm(x, shape[3], w, b, eps=EPS, activation=activation)
        first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        d = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, activation, gy.detach())
        for outs, cots in (((0,), (v, None, None)), ((0, 1, 2), (v, vw, vb)), ((1,), (0 * v, vw, None)),
                           ((1, 2), (0 * v, vw, vb))):
            got = torch.autograd.grad([first[i] for i in outs], (x, gy, w, b), [cots[i] for i in outs], retain_graph=True,
                                      allow_unused=True)
            ref, sizes = d.second(*cots)
            _close(got[0], ref[0], SECOND[dtype], "dx'")
            _close(got[1], ref[1], SECOND[dtype], "dg'")
            for k in (2, 3):
                if got[k] is not None:
                    _close_sum(got[k], ref[k], sizes[k - 2], "dw'" if k == 2 else "db'")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(20011, 1, 64, 8), (30000, 1, 30, 5), (5003, 9, 64, 8), (3001, 70, 40, 5),
                                   (1, 131072, 32, 4), (4, 9001, 72, 3), (2003, 1, 4096, 1),
                                   (1, 131072, 65, 13), (500, 1000, 30, 5), (1030, 130, 63, 63), (21, 1999, 330, 11),
                                   (3001, 401, 7, 7), (37, 4001, 60, 2)])
def test_larger(device, shape, dtype):
    from ictc_o3 import group_norm
    x, w, b, gy, v, vw, vb = _inputs(shape, dtype, device)
    for t in (x, w, b, gy):
        t.requires_grad_()
    d = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, "silu", gy.detach())
    runs = []
    for _ in range(2):
        y = group_norm(x, shape[3], w, b, eps=EPS, activation="silu")
        first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        runs.append((y, *first, *torch.autograd.grad(first, (x, gy, w, b), (v, vw, vb))))
    assert all(torch.equal(i, j) for i, j in zip(*runs))       # a fixed order of every sum
    y, dx, dw, db, *second = runs[0]
    _close(y, definition(x.detach().double(), shape[3], w.detach().double(), b.detach().double(), EPS, "silu"), TOL[dtype],
           "y")
    ref, sizes = d.first()
    _close(dx, ref[0], TOL[dtype], "dx")
    _close_sum(dw, ref[1], sizes[0], "dw")
    _close_sum(db, ref[2], sizes[1], "db")
    ref, sizes = d.second(v, vw, vb)
    _close(second[0], ref[0], SECOND[dtype], "dx'")
    _close(second[1], ref[1], SECOND[dtype], "dg'")
    _close_sum(second[2], ref[2], sizes[0], "dw'")
    _close_sum(second[3], ref[3], sizes[1], "db'")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(37, 1, 64, 8), (9, 1, 35, 5), (5, 1, 600, 200), (3, 1, 2176, 1), (7, 9, 64, 8),
                                   (5, 33, 30, 5), (2, 257, 330, 11), (3, 300, 64, 8), (2, 4099, 30, 5), (1, 700, 2304, 1),
                                   (9, 1, 384, 3), (9, 1, 392, 4), (0, 1, 16, 4),
                                   (700, 1, 16, 4), (11, 1, 128, 1), (37, 1, 256, 8), (1030, 1, 512, 64), (5, 1, 1024, 2),
                                   (3, 1, 2048, 2), (6, 1, 768, 2), (9, 1, 640, 40), (4, 1, 2048, 256), (3, 1, 96, 3),
                                   (1, 131072, 65, 13), (501, 1000, 30, 5), (2100, 65, 130, 26), (9, 1, 999, 3),
                                   (5, 3, 77, 7)])
def test_x_in_8_bits(device, shape, dtype):
    """The result is that of whole rows, bit for bit; the derivatives are the formulas at the decoded x."""
    from ictc_o3 import decode_activations, encode_activations, group_norm
    x, w, b, gy, v, vw, vb = _inputs(shape, dtype, device)
    value = decode_activations(*encode_activations(x), dtype=dtype)
    for t in (x, w, b, gy):
        t.requires_grad_()
    for activation in (None, "silu"):
        y = group_norm(x, shape[3], w, b, eps=EPS, activation=activation, save_bits=8)
        assert torch.equal(y, group_norm(x, shape[3], w, b, eps=EPS, activation=activation))
        got = torch.autograd.grad(y, (x, w, b), gy, retain_graph=True)
        first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        assert all(torch.equal(i, j) for i, j in zip(got, first))
        if not x.numel():
            assert (got[1] == 0).all() and (got[2] == 0).all()
            continue
        d = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, activation, gy.detach(), value)
        ref, sizes = d.first()
        _close(got[0], ref[0], TOL[dtype], "dx")
        _close_sum(got[1], ref[1], sizes[0], "dw")
        _close_sum(got[2], ref[2], sizes[1], "db")
        second = torch.autograd.grad(first, (x, gy, w, b), (v, vw, vb), allow_unused=True)
        ref, sizes = d.second(v, vw, vb)
        _close(second[0], ref[0], SECOND[dtype], "dx'")
        _close(second[1], ref[1], SECOND[dtype], "dg'")
        _close_sum(second[2], ref[2], sizes[0], "dw'")
        if second[3] is not None:
            _close_sum(second[3], ref[3], sizes[1], "db'")


def test_8_bits_keep_a_byte_an_element(device):
    from ictc_o3 import group_norm
    base = torch.randn(16384, 16, 64, device=device, requires_grad=True)

    def kept(bits):
        before = torch.cuda.memory_allocated()
        y = group_norm(base * 2.0, 8, activation="silu", save_bits=bits)
        return torch.cuda.memory_allocated() - before - y.numel() * 4

    stats = 16384 * 8 * 8
    assert kept(None) > base.numel() * 4 and kept(8) < base.numel() * (1 + 4 / 64) + stats + (1 << 20)


def test_absent_parameters_and_partial_gradients(device):
    from ictc_o3 import group_norm
    for shape in ((19, 1, 96, 4), (3, 300, 24, 2), (1, 6000, 24, 2)):
        x, w, b, gy, v, *_ = _inputs(shape, torch.float32, device, 3)
        for use_w, use_b in ((False, False), (True, False), (False, True)):
            ww, bb = w if use_w else None, b if use_b else None
            xr = x.clone().requires_grad_()
            y = group_norm(xr, shape[3], ww, bb, eps=EPS, activation="silu")
            (gx,) = torch.autograd.grad(y, xr, gy, create_graph=True)
            (gxx,) = torch.autograd.grad(gx, xr, v)
            d = Derivatives(x, shape[3], ww, bb, EPS, "silu", gy)
            _close(gx, d.first()[0][0], 1e-5, "dx")
            _close(gxx, d.second(v)[0][0], 4e-5, "dx'")
        for k, p in enumerate((w, b)):
            p = p.clone().requires_grad_()
            args = (p, b) if k == 0 else (w, p)
            (got,) = torch.autograd.grad(group_norm(x, shape[3], *args, eps=EPS, activation="silu"), p, gy)
            ref, sizes = Derivatives(x, shape[3], w, b, EPS, "silu", gy).first()
            _close_sum(got, ref[1 + k], sizes[k], "dw or db")


def test_against_differences(device):
    """Central differences of the kernel's own output at step h: the truncation h^2 f'''/6 and the rounding
    2^-23 sqrt(terms) / h are both under 1e-3 of the gradient's norm at h = 2^-6; the bound is 1e-2."""
    from ictc_o3 import group_norm
    for shape in ((5, 1, 40, 4), (2, 300, 12, 3)):
        x, w, b, gy, *_ = _inputs(shape, torch.float32, device, 9)
        h = 2.0 ** -6
        args = [t.requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(group_norm(args[0], shape[3], *args[1:], activation="silu"), args, gy)
        for i in range(3):
            step = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(device)
            out = []
            for sign in (1, -1):
                moved = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(args)]
                out.append((group_norm(moved[0], shape[3], *moved[1:], activation="silu").double() * gy.double()).sum())
            slope = (grads[i].double() * step.double()).sum()
            assert ((out[0] - out[1]) / (2 * h) - slope).abs() < 1e-2 * grads[i].double().norm() * step.double().norm()


def test_strides_and_axes(device):
    from ictc_o3 import group_norm
    x, w, b, gy, *_ = _inputs((4, 30, 24, 3), torch.bfloat16, device, 4)
    plain = group_norm(x, 3, w, b)
    assert torch.equal(group_norm(x.view(4, 5, 6, 24), 3, w, b), plain.view(4, 5, 6, 24))
    wide = torch.zeros(4, 30, 31, dtype=torch.bfloat16, device=device)
    wide[..., 3:27] = x
    assert torch.equal(group_norm(wide[..., 3:27], 3, w, b), plain)
    assert torch.equal(group_norm(x.transpose(0, 1).contiguous().transpose(0, 1), 3, w, b), plain)
    assert torch.equal(group_norm(x.permute(0, 2, 1).contiguous().permute(0, 2, 1), 3, w, b), plain)   # channels first
    assert torch.equal(group_norm(x[:1].expand(4, 30, 24), 3, w, b), plain[:1].expand(4, 30, 24))
    assert torch.equal(group_norm(x[::2], 3, w, b), plain[::2])
    xr = wide.clone().requires_grad_()
    (got,) = torch.autograd.grad(group_norm(xr[..., 3:27], 3, w, b), xr, gy.permute(0, 2, 1).contiguous().permute(0, 2, 1))
    xr = x.clone().requires_grad_()
    (ref,) = torch.autograd.grad(group_norm(xr, 3, w, b), xr, gy)
    assert torch.equal(got[..., 3:27], ref) and (got[..., :3] == 0).all()
    (summed,) = torch.autograd.grad(group_norm(xr, 3, w, b).sum(), xr)                 # a gradient of stride zero
    (ones,) = torch.autograd.grad(group_norm(xr, 3, w, b), xr, torch.ones_like(x))
    assert torch.equal(summed, ones)


@pytest.mark.parametrize("shape", [(40, 1, 64, 8), (40, 6, 32, 4), (5, 300, 32, 4), (2, 9000, 16, 2)])
def test_far_means_and_values_of_one_size(device, shape):
    """A mean 4,096 times the spread: x itself keeps 12 of FP32's 24 bits of it, and no more is lost (bound: 64 units of
    2^-24 of the mean over the spread, 1.6e-2).  Samples of one value have no spread: y is the bias, exactly."""
    from ictc_o3 import group_norm
    x, w, b, *_ = _inputs(shape, torch.float32, device)
    far = 4096 + torch.round(x * 1024) / 1024
    assert rel_err(group_norm(far, shape[3]), definition(far.double(), shape[3], None, None, EPS, None)) < 1.6e-2
    assert torch.equal(group_norm(torch.full_like(x, 2.5), shape[3], w, b), b.expand(x.shape))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(40, 1, 64, 8), (40, 6, 32, 4), (40, 300, 32, 4), (40, 9000, 16, 2), (40, 1, 2176, 1)])
def test_samples_whose_squares_leave_the_range(device, shape, dtype):
    """Finite samples spread over up to 2^110, whose variance FP32 does not hold, beside ordinary ones: a power of two
    changes no rounding, so the bounds are the ordinary ones, sample by sample."""
    from ictc_o3 import group_norm
    x, w, b, gy, *_ = _inputs(shape, dtype, device, 3)
    size = torch.exp2(torch.tensor([0.0, 62.0, 66.0, 90.0, 110.0], device=device)).repeat(8).view(-1, *[1] * (x.dim() - 1))
    x = (x.float() * size).to(dtype).requires_grad_()
    y = group_norm(x, shape[3], w, b, activation="silu")
    (gx,) = torch.autograd.grad(y, x, gy)
    _close(y, definition(x.detach().double(), shape[3], w.double(), b.double(), EPS, "silu"), TOL[dtype], "y")
    ref = Derivatives(x.detach(), shape[3], w, b, EPS, "silu", gy).first()[0][0]
    _close(gx.double() * size, ref * size, TOL[dtype], "dx")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(40, 9, 32, 4), (40, 3, 35, 5), (9, 1, 36, 3), (7, 9, 64, 8), (33, 301, 32, 4),
                                   (3, 300, 30, 5), (2, 9001, 16, 2)])
def test_samples_of_one_large_value(device, shape, dtype):
    """2^121 everywhere: means and deviations are exact, so the bounds are the ordinary ones; the mean over the deviation
    is past FP32, which lanes and positions that hold nothing must not see."""
    from ictc_o3 import group_norm
    x, w, b, gy, v, vw, vb = _inputs(shape, dtype, device, 5)
    x = torch.full_like(x, 2.0 ** 121)
    for t in (x, w, b, gy):
        t.requires_grad_()
    y = group_norm(x, shape[3], w, b, eps=EPS, activation="silu")
    first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
    second = torch.autograd.grad(first, (x, gy, w, b), (v, vw, vb))
    d = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, "silu", gy.detach())
    (dx, dw, db), (sw, sb) = d.first()
    ref, sizes = d.second(v, vw, vb)
    _close(y, torch.nn.functional.silu(b.double()).expand(x.shape), TOL[dtype], "y")
    _close(first[0], dx, TOL[dtype], "dx")
    _close_sum(first[1], dw, sw, "dw")
    _close_sum(first[2], db, sb, "db")
    _close(second[0], ref[0], SECOND[dtype], "dx'")
    _close(second[1], ref[1], SECOND[dtype], "dg'")
    _close_sum(second[2], ref[2], sizes[0], "dw'")
    _close_sum(second[3], ref[3], sizes[1], "db'")


@pytest.mark.parametrize("shape", [(33, 1, 64, 8), (33, 6, 32, 4), (33, 300, 32, 4), (33, 5000, 16, 2), (33, 1, 2176, 1)])
def test_nan_and_infinity_stay_in_their_group(device, shape):
    from ictc_o3 import group_norm
    x, w, b, gy, *_ = _inputs(shape, torch.float32, device, 2)
    clean = group_norm(x, shape[3], w, b, activation="silu")
    flat = x.view(33, -1)
    flat[4, 0], flat[20, -1] = float("nan"), float("inf")
    bad = torch.zeros(33, shape[1], shape[3], shape[2] // shape[3], dtype=torch.bool, device=device)
    bad[4, :, 0], bad[20, :, -1] = True, True
    bad = bad.view(x.shape)
    x.requires_grad_()
    y = group_norm(x, shape[3], w, b, activation="silu")
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])
    (gx,) = torch.autograd.grad(y, x, gy)
    assert torch.isnan(gx[bad]).all() and torch.isfinite(gx[~bad]).all()


def test_large_arguments_of_the_activation(device):
    from ictc_o3 import group_norm
    x, w, b, gy, v, *_ = _inputs((8, 1, 32, 2), torch.float32, device)
    b = torch.linspace(-200, 200, 32, device=device)
    x.requires_grad_()
    y = group_norm(x, 2, w, b, eps=EPS, activation="silu")
    (gx,) = torch.autograd.grad(y, x, gy, create_graph=True)
    (gxx,) = torch.autograd.grad(gx, x, v)
    d = Derivatives(x.detach(), 2, w, b, EPS, "silu", gy)
    _close(y, definition(x.detach().double(), 2, w.double(), b.double(), EPS, "silu"), 1e-5, "y")
    _close(gx, d.first()[0][0], 1e-5, "dx")
    _close(gxx, d.second(v)[0][0], 4e-5, "dx'")


def test_third_derivative_raises(device):
    from ictc_o3 import group_norm
    for bits in (None, 8):
        x = torch.randn(4, 32, device=device, requires_grad=True)
        (g1,) = torch.autograd.grad(group_norm(x, 4, save_bits=bits).square().sum(), x, create_graph=True)
        (g2,) = torch.autograd.grad(g1.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="third"):
            torch.autograd.grad(g2.sum(), x)


@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("shape", [(300, 1, 64, 8), (5, 300, 32, 4), (1, 9000, 64, 4)])
def test_streams_and_graph_replays(device, shape, bits):
    from ictc_o3 import group_norm
    x, w, b, gy, v, *_ = _inputs(shape, torch.float32, device, 8)
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        y = group_norm(x, shape[3], w, b, activation="silu", save_bits=bits)
        first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        second = torch.autograd.grad(first[0], (x, w), v)
        return [t.detach() for t in (y, *first, *second)]

    here = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(i, j) for i, j in zip(here, there))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.mul_(-1.25).add_(0.25)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) for i, j in zip(held, eager)), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(77, 1, 130, 10), (7, 300, 12, 3), (1, 9000, 12, 3)])
def test_the_same_without_a_graph(device, shape, dtype):
    from ictc_o3 import group_norm
    x, w, b, *_ = _inputs(shape, dtype, device, 5)
    plain = group_norm(x, shape[3], w, b, activation="silu")
    kept = group_norm(x, shape[3], w.clone().requires_grad_(), b, activation="silu")
    with torch.no_grad():
        off = group_norm(x.clone().requires_grad_(), shape[3], w, b, activation="silu")
    with torch.inference_mode():
        inference = group_norm(x, shape[3], w, b, activation="silu", save_bits=8)
    assert kept.requires_grad and not plain.requires_grad and not off.requires_grad
    assert all(torch.equal(t, kept) for t in (plain, off, inference))


def test_refusals(device):
    from ictc_o3 import group_norm
    x, w = torch.zeros(4, 12, device=device), torch.ones(12, device=device)
    for call, match in ((lambda: group_norm(x.double(), 2), "float32"), (lambda: group_norm(x[0], 2), "shape"),
                        (lambda: group_norm(x[:, :0], 1), "channels"), (lambda: group_norm(x, 5), "divide"),
                        (lambda: group_norm(x, 0), "divide"), (lambda: group_norm(x, 2, w[:6]), "shape"),
                        (lambda: group_norm(x, 2, w.bfloat16()), "type"), (lambda: group_norm(x, 2, w, w.cpu()), "device"),
                        (lambda: group_norm(x, 2, eps=-1.0), "eps"), (lambda: group_norm(x, 2, eps=float("nan")), "eps"),
                        (lambda: group_norm(x, 2, activation="relu"), "activation"),
                        (lambda: group_norm(x, 2, save_bits=4), "save_bits")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError):      # x changed between the passes
        xr = torch.randn(4, 12, device=device, requires_grad=True)
        t = xr * 1.0
        y = group_norm(t, 2)
        t.add_(1)
        y.sum().backward()


def test_offsets_past_32_bits(device):
    """More than 2^31 elements, as many rows and as one sample: the first and last rows and the sums."""
    from ictc_o3 import group_norm
    N, C = 34000000, 64
    g = torch.Generator(device).manual_seed(1)
    x = torch.randn(N, C, device=device, generator=g, dtype=torch.bfloat16)
    ends = torch.cat([torch.arange(0, 200, device=device), torch.arange(N - 200, N, device=device)])
    gy = torch.zeros(N, C, device=device, dtype=torch.bfloat16)
    gy[ends] = torch.randn(400, C, device=device, generator=g).bfloat16()
    for bits in (None, 8):
        xr, w = x.detach().requires_grad_(), torch.ones(C, device=device, dtype=torch.bfloat16, requires_grad=True)
        y = group_norm(xr, 8, w, activation="silu", save_bits=bits)
        gx, gw = torch.autograd.grad(y, (xr, w), gy)
        few, fw = x[ends].double().requires_grad_(), torch.ones(C, device=device, dtype=torch.float64, requires_grad=True)
        Y = definition(few, 8, fw, None, EPS, "silu")
        ref = torch.autograd.grad(Y, (few, fw), gy[ends].double())
        assert rel_err(y[ends], Y) < TOL[torch.bfloat16]
        if bits is None:
            assert rel_err(gx[ends], ref[0]) < TOL[torch.bfloat16] and rel_err(gw, ref[1]) < TOL[torch.bfloat16]
        else:      # (x off by 1/254 of a row's largest at most, about 3 of 64: a few hundredths of a gradient)
            assert rel_err(gx[ends], ref[0]) < 0.1 and rel_err(gw, ref[1]) < 0.1
        assert (gx[1000:200000] == 0).all()
        del y, gx, xr
    one = x.view(1, N, C)
    y = group_norm(one, 8)
    X = one.view(N, 8, 8)
    count, sums, squares = N * 8, 0, 0
    for part in X.split(1 << 22):
        sums, squares = sums + part.double().sum((0, 2)), squares + part.double().square().sum((0, 2))
    mean = sums / count
    r = 1 / torch.sqrt(squares / count - mean ** 2 + EPS)
    ref = (X[ends].double() - mean[:, None]) * r[:, None]
    assert rel_err(y.view(N, 8, 8)[ends], ref) < TOL[torch.bfloat16]


@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1030, 130, 63, 63), (3001, 401, 7, 7), (501, 1001, 30, 15), (1, 131072, 65, 13)])
def test_samples_of_one_large_value_in_many_small_groups(device, shape, dtype, bits):
    """2^121 everywhere, as in the test of one large value, where a tile's chunks reach over groups; 127 (2^121 / 127), which
    its codes stand for, is 2^121 again."""
    from ictc_o3 import decode_activations, encode_activations, group_norm
    x, w, b, gy, *_ = _inputs(shape, dtype, device, 5)
    x = torch.full_like(x, 2.0 ** 121)
    assert torch.equal(decode_activations(*encode_activations(x), dtype=dtype), x)
    for t in (x, w, b):
        t.requires_grad_()
    for activation in (None, "silu"):
        y = group_norm(x, shape[3], w, b, eps=EPS, activation=activation, save_bits=bits)
        first = torch.autograd.grad(y, (x, w, b), gy)
        ref, sizes = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, activation, gy).first()
        z = b.detach().double()
        _close(y, (torch.nn.functional.silu(z) if activation else z).expand(x.shape), TOL[dtype], "y")
        _close(first[0], ref[0], TOL[dtype], "dx")
        _close_sum(first[1], ref[1], sizes[0], "dw")
        _close_sum(first[2], ref[2], sizes[1], "db")


@pytest.mark.parametrize("spread", [2.0 ** -12, 2.0 ** -17, 2.0 ** -20])
@pytest.mark.parametrize("shape", [(40, 1, 64, 8), (33, 1, 60, 5), (3, 1, 8192, 1), (40, 6, 32, 4), (9, 5, 45, 5),
                                   (40, 300, 32, 4), (3, 513, 5, 5), (1, 9000, 16, 2), (1, 131072, 64, 64),
                                   (1, 700, 2304, 1), (3001, 401, 7, 7), (1, 131072, 65, 13)])
def test_means_far_from_zero_as_near_ones(device, shape, spread):
    """Means of up to 2^20 deviations, in every form and pass.  x less its mean is as exact as x is: less the mean in FP32
    without an error (the operands are within a factor of two), less what that rounding left with one of half a unit of
    the result.  So the bounds are the ordinary ones, and those of sums count h itself and not x and the mean; ga
    depends on h by the activation, with a slope of at most 1/2."""
    from ictc_o3 import group_norm
    x, w, b, gy, v, vw, vb = _inputs(shape, torch.float32, device, 6)
    x = x + 1.2345 / spread * (1 + torch.rand(shape[0], *[1] * (x.dim() - 1), device=device,
                                               generator=torch.Generator(device).manual_seed(3)))
    for t in (x, w, b, gy):
        t.requires_grad_()
    for activation in (None, "silu"):
        y = group_norm(x, shape[3], w, b, eps=EPS, activation=activation)
        first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        second = torch.autograd.grad(first, (x, gy, w, b), (v, vw, vb), allow_unused=True)
        d = Derivatives(x.detach(), shape[3], w.detach(), b.detach(), EPS, activation, gy.detach())
        ref, _ = d.first()
        _close(y, definition(x.detach().double(), shape[3], w.detach().double(), b.detach().double(), EPS, activation), 1e-5,
               "y")
        _close(first[0], ref[0], 1e-5, "dx")
        size = d.g.abs() * (1.1 + d.h.abs() / 2)
        _close_sum(first[1], ref[1], d._channels(size * (1 + d.h.abs())), "dw")
        _close_sum(first[2], ref[2], d._channels(size), "db")
        ref, _ = d.second(v, vw, vb)
        _close(second[0], ref[0], 4e-5, "dx'")
        _close(second[1], ref[1], 4e-5, "dg'")


@pytest.mark.parametrize("shape", [(40, 1, 64, 8), (40, 300, 32, 4), (1, 9000, 16, 2), (1, 131072, 64, 64)])
def test_one_value_of_a_mean(device, shape):
    """The entry points without the means' rest: the same output; gradients off by half a unit of the mean in h."""
    from ictc_o3 import _native as nat
    from ictc_o3 import group_norm
    samples, positions, channels, groups = shape
    x, w, b, gy, *_ = _inputs(shape, torch.float32, device, 6)
    x = (x + 100.0).requires_grad_()
    y = group_norm(x, groups, w, b, eps=EPS, activation="silu")
    (dx,) = torch.autograd.grad(y, x, gy)
    mean, rstd = torch.empty(2, samples, groups, device=device)
    out, got = torch.empty_like(x), torch.empty_like(x)
    size = nat.lib().ictc_group_norm_workspace_bytes
    sizes = [size(0, k, samples, positions, channels, groups) for k in (0, 1)]
    ws = torch.empty(max(*sizes, 8), dtype=torch.uint8, device=device)
    at = (samples, positions, channels, groups, w.data_ptr(), b.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    nat.call("ictc_group_norm_fwd", 0, x.data_ptr(), *at, EPS, 1, out.data_ptr(), mean.data_ptr(), rstd.data_ptr(), None, None,
             ws.data_ptr(), sizes[0], stream)
    nat.call("ictc_group_norm_bwd", 0, x.data_ptr(), None, None, gy.data_ptr(), *at, 1, mean.data_ptr(), rstd.data_ptr(),
             got.data_ptr(), None, None, ws.data_ptr(), sizes[1], stream)
    X = x.detach().double().view(samples, -1, groups, channels // groups)
    assert torch.equal(out, y) and rel_err(mean, X.mean((1, 3))) < 2.0 ** -23
    # half a unit of the mean times r, in h and with a slope of two or less in all that follows; and the ordinary bound
    assert rel_err(got, dx.double()) < 1e-5 + 2 * 2.0 ** -25 * (X.mean((1, 3)).abs() * rstd).max() * 4


@pytest.mark.parametrize("shape", [(300, 1, 64, 8), (9, 5, 45, 5), (40, 300, 32, 4), (1, 9000, 160, 2), (501, 1000, 30, 5)])
@pytest.mark.parametrize("far", [0.0, 3.0, 30.0])
def test_error_of_gradients_from_8_bits(device, shape, far):
    """What is promised of x kept in 8 bits: h is off by at most half a scale (1/254 of the largest magnitude of its block of
    128 channels) times r, so without an activation dw is off by as much of each of its terms, and dx by r (|eh| <u h> +
    |h| <u eh>) with both h's; and by the ordinary bounds."""
    from ictc_o3 import encode_activations, group_norm
    x, w, b, gy, *_ = _inputs(shape, torch.float32, device, 4)
    x = x + far
    scales = encode_activations(x)[1].double().repeat_interleave(128, -1)[..., :shape[2]]
    x, w = x.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(group_norm(x, shape[3], w, b, eps=EPS, save_bits=8), (x, w), gy)
    d = Derivatives(x.detach(), shape[3], w.detach(), b, EPS, None, gy)
    (dx, dw, _), (sw, _) = d.first()
    off = (scales * (0.5 + 127 * 2.0 ** -21)).view(d.h.shape) * d.r
    mean = lambda t: t.abs().mean((1, 3), keepdim=True)
    u = d.ga * d.w
    bound = d.r * (off * (mean(u * d.h) + mean(u * off)) + d.h.abs() * mean(u * off))
    assert ((got[1].double() - dw).abs() <= d._channels(d.ga.abs() * off) + 600 * 2.0 ** -24 * (sw + d._channels(d.ga.abs() * off))).all()
    assert ((got[0].double() - dx).abs() <= bound.view(x.shape) + 1e-5 * (dx.abs().max() + bound.max())).all()
