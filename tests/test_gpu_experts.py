"""Per-row expert linears against their formula in float64: output, gradients, gradients of gradients, differences,
odd sizes and layouts, empty experts, rows of no expert, refusals.

Bounds (max-norm, relative to the largest reference value): a result adds K terms in FP32 (K the inputs, or the rows of
an expert for the weights' gradient) by matrix instructions over 32 of them and a running sum, so its error is at most
K / 32 + 32 units of 2^-24 of the sum of magnitudes; with random signs the sum of magnitudes is about sqrt(K) times the
result and the roundings add like their square root: under (sqrt(K / 32) + 6) sqrt(K) 2^-24 relative to a typical
result, and the largest result is three or more times a typical one.  For K up to 4,096 that is 1.4e-5; the bound is
2e-5.  bfloat16 and float16 results are rounded once more: 2^-9 and 2^-11, the bounds are twice that.
"""
import math

import pytest
import torch

from helpers import rel_err

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 2e-5, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _formula(x, W, b, ids):
    keep = ((ids >= 0) & (ids < W.shape[0])).nonzero().view(-1)
    y = torch.zeros(x.shape[0], W.shape[1], dtype=x.dtype, device=x.device)
    parts = []
    for e in range(W.shape[0]):
        at = (ids == e).nonzero().view(-1)
        z = x[at] @ W[e].t()
        parts.append((at, z if b is None else z + b[e]))
    order = torch.cat([at for at, _ in parts])
    assert order.numel() == keep.numel()
    return y.index_copy(0, order, torch.cat([z for _, z in parts]))


def _inputs(rows, experts, K, M, dtype, seed, device, bad=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (rows,), generator=g)
    if experts > 2:
        ids[ids == 1] = 2                                  # an expert without rows
    if bad and rows > 4:
        ids[1], ids[rows - 1] = -1, experts + 3            # rows of no expert
    x = torch.randn(rows, K, generator=g).to(dtype)
    W = (torch.randn(experts, M, K, generator=g) / math.sqrt(K)).to(dtype)
    b = torch.randn(experts, M, generator=g).to(dtype)
    gy = torch.randn(rows, M, generator=g).to(dtype)
    return tuple(t.to(device) for t in (ids, x, W, b, gy))


def _check(got, ref, names):
    for a, r, name in zip(got, ref, names):
        assert torch.isfinite(a).all() and a.shape == r.shape, name
        assert rel_err(a, r) < TOL[a.dtype], (name, rel_err(a, r))


def _run(ids, x, W, b, gy, create=False):
    from ictc_o3 import expert_linear, expert_order
    args = [t.detach().requires_grad_() for t in (x, W, b)]
    y = expert_linear(args[0], args[1], expert_order(ids, W.shape[0]), args[2])
    return args, y, torch.autograd.grad(y, args, gy, create_graph=create)


def _reference(ids, x, W, b, gy):
    args = [t.detach().double().requires_grad_() for t in (x, W, b)]
    y = _formula(*args, ids)
    return args, y, torch.autograd.grad(y, args, gy.double(), create_graph=True)


SHAPES = [(1, 1, 1, 1), (3, 2, 5, 7), (130, 4, 64, 64), (257, 3, 33, 129), (1000, 10, 128, 128), (700, 89, 200, 333),
          (2000, 5, 96, 1), (900, 7, 1, 160), (515, 1, 256, 255), (1500, 70, 127, 16), (4000, 3, 144, 272),
          (40000, 9, 80, 24), (33000, 6, 257, 40), (1, 8, 1024, 300), (40, 3, 1000, 130), (200, 60, 520, 136), (17, 2, 77, 33)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,K,M", SHAPES)
def test_output_and_gradients(device, rows, experts, K, M, dtype):
    data = _inputs(rows, experts, K, M, dtype, rows + K, device)
    _, y, got = _run(*data)
    _, Y, ref = _reference(*data)
    _check((y, *got), (Y, *ref), ("y", "gx", "gW", "gb"))
    if experts > 2:
        assert got[1][1].abs().max() == 0 and got[2][1].abs().max() == 0
    if rows > 4:
        assert y[1].abs().max() == 0 and got[0][rows - 1].abs().max() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,K,M", [(9000, 4, 72, 200), (20000, 2, 64, 136), (6000, 90, 64, 64)])
def test_many_rows_repeat_bit_by_bit(device, rows, experts, K, M, dtype):
    """Experts of several runs in the weights' gradient, whose partial sums are added in order."""
    data = _inputs(rows, experts, K, M, dtype, 11, device)
    _, y, got = _run(*data)
    _, Y, ref = _reference(*data)
    _check((y, *got), (Y, *ref), ("y", "gx", "gW", "gb"))
    _, y2, again = _run(*data)
    assert torch.equal(y, y2) and all(torch.equal(i, j) for i, j in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("rows,experts,K,M", [(30000, 5, 9, 131), (30000, 3, 131, 9), (30000, 4, 65, 193), (20000, 3, 8, 300),
                                              (30000, 2, 300, 7), (26000, 3, 127, 130), (18000, 2, 200, 15)])
def test_rows_that_end_inside_a_chunk(device, rows, experts, K, M, dtype):
    """Many rows whose ends, beginnings and pitches are no multiples of 16 bytes, between NaN."""
    from ictc_o3 import expert_linear, expert_order
    ids, x, W, b, gy = _inputs(rows, experts, K, M, dtype, rows + K, device)
    _, Y, ref = _reference(ids, x, W, b, gy)
    order = expert_order(ids, experts)
    for front in (0, 3):
        def held(t):
            wide = torch.full((rows, t.shape[1] + front + 4), float("nan"), dtype=dtype, device=device)
            wide[:, front:front + t.shape[1]] = t
            return wide[:, front:front + t.shape[1]]
        args = [held(x).requires_grad_(), W.clone().requires_grad_(), b.clone().requires_grad_()]
        y = expert_linear(args[0], args[1], order, args[2])
        _check((y, *torch.autograd.grad(y, args, held(gy))), (Y, *ref), ("y", "gx", "gW", "gb"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_gradients(device, dtype):
    data = _inputs(300, 4, 40, 72, dtype, 2, device)
    args, y, first = _run(*data, create=True)
    Args, Y, First = _reference(*data)
    g = torch.Generator().manual_seed(3)
    v = [torch.randn(t.shape, generator=g).to(dtype).to(device) for t in first]
    for outs, wrt in (((0,), (1,)), ((1,), (0,)), ((0, 1), (0, 1))):
        got = torch.autograd.grad([first[i] for i in outs], [args[i] for i in wrt], [v[i] for i in outs],
                                  retain_graph=True, create_graph=True)
        ref = torch.autograd.grad([First[i] for i in outs], [Args[i] for i in wrt], [v[i].double() for i in outs],
                                  retain_graph=True, create_graph=True)
        if dtype is torch.float32 or len(outs) == 1:
            _check(got, ref, [f"{outs} by {i}" for i in wrt])


def test_gradient_of_the_output_gradient(device):
    """d/d gy of <v, gx> + <V, gW> + <c, gb>, and with the bias gradient alone."""
    ids, x, W, b, gy = _inputs(200, 3, 24, 40, torch.float32, 5, device)
    from ictc_o3 import expert_linear, expert_order
    order = expert_order(ids, 3)
    g = torch.Generator().manual_seed(1)
    for kind in ("own", "double"):
        f = (lambda t: t.clone().requires_grad_()) if kind == "own" else (lambda t: t.double().requires_grad_())
        a = [f(t) for t in (x, W, b, gy)]
        y = expert_linear(a[0], a[1], order, a[2]) if kind == "own" else _formula(*a[:3], ids)
        first = torch.autograd.grad(y, a[:3], a[3], create_graph=True)
        g.manual_seed(1)
        v = [torch.randn(t.shape, generator=g).to(t.dtype).to(device) for t in first]
        second = torch.autograd.grad(first, a[3], v, retain_graph=True)
        bias_only = torch.autograd.grad(first[2], a[3], v[2])
        if kind == "own":
            mine = (*second, *bias_only)
        else:
            _check(mine, (*second, *bias_only), ("all", "bias"))


def test_against_differences(device):
    """The output is linear in each argument, so a central difference at step 1 has only roundings: 2^-23 times the
    values' norm over the slope's, under 1e-4; the bound is 1e-3."""
    from ictc_o3 import expert_linear, expert_order
    ids, x, W, b, gy = _inputs(60, 4, 30, 50, torch.float32, 6, device)
    order = expert_order(ids, 4)
    args, _, grads = _run(ids, x, W, b, gy)
    for i in range(3):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).to(device)
        out = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * d if j == i else 0) for j, t in enumerate(args)]
            out.append((expert_linear(moved[0], moved[1], order, moved[2]).double() * gy.double()).sum())
        slope = (grads[i].double() * d.double()).sum()
        assert ((out[0] - out[1]) / 2 - slope).abs() < 1e-3 * grads[i].double().norm() * d.double().norm()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_odd_bases(device, dtype):
    from ictc_o3 import expert_linear, expert_order
    ids, x, W, b, gy = _inputs(300, 3, 70, 90, dtype, 7, device)
    order = expert_order(ids, 3)
    plain = expert_linear(x, W, order, b)
    wide = torch.full((300, 101), float("nan"), dtype=dtype, device=device)
    wide[:, 5:75] = x                                          # odd pitch and offset between NaN
    assert torch.equal(expert_linear(wide[:, 5:75], W, order, b), plain)
    assert torch.equal(expert_linear(x.t().contiguous().t(), W, order, b), plain)
    flat = torch.empty(W.numel() + 1, dtype=dtype, device=device)
    flat[1:] = W.flatten()
    assert torch.equal(expert_linear(x, flat[1:].view(W.shape), order, b), plain)
    assert torch.equal(expert_linear(x, W.transpose(1, 2).contiguous().transpose(1, 2), order, b), plain)
    row = x[:1].expand(300, 70)                                # row pitch zero
    assert torch.equal(expert_linear(row, W, order, b), expert_linear(row.contiguous(), W, order, b))
    xr, Wr = x.clone().requires_grad_(), W.clone().requires_grad_()
    broad = torch.autograd.grad(expert_linear(xr, Wr, order, b), (xr, Wr), gy[:, :1].expand(300, 90), retain_graph=True)
    whole = torch.autograd.grad(expert_linear(xr, Wr, order, b), (xr, Wr), gy[:, :1].expand(300, 90).contiguous())
    assert all(torch.equal(i, j) for i, j in zip(broad, whole))


def test_no_rows_and_no_valid_rows(device):
    from ictc_o3 import expert_linear, expert_order
    for rows in (0, 300):
        ids = torch.full((rows,), 9, dtype=torch.int64, device=device)
        x = torch.randn(rows, 20, device=device, requires_grad=True)
        W = torch.randn(3, 30, 20, device=device, requires_grad=True)
        b = torch.randn(3, 30, device=device, requires_grad=True)
        y = expert_linear(x, W, expert_order(ids, 3), b)
        grads = torch.autograd.grad(y, (x, W, b), torch.ones_like(y))
        assert y.shape == (rows, 30)
        for t in (y, *grads):
            assert t.numel() == 0 or t.abs().max() == 0


def test_nan_stays_in_its_row(device):
    from ictc_o3 import expert_linear, expert_order
    for dtype in TYPES:
        ids, x, W, b, _ = _inputs(400, 3, 100, 60, dtype, 8, device)
        order = expert_order(ids, 3)
        clean = expert_linear(x, W, order, b)
        x[7, 99], x[250, 0] = float("nan"), float("inf")
        y = expert_linear(x, W, order, b)
        bad = torch.zeros(400, dtype=torch.bool, device=device)
        bad[[7, 250]] = True
        assert torch.isnan(y[7]).all() and not torch.isfinite(y[250]).any() and torch.equal(y[~bad], clean[~bad])


def test_same_as_the_species_linear(device):
    """The square FP32 species linear that the model uses computes the same map."""
    from ictc_o3 import expert_linear, expert_order
    from ictc_o3.ops.linear import species_linear
    ids, x, W, _, _ = _inputs(1000, 10, 128, 128, torch.float32, 9, device)
    assert rel_err(expert_linear(x, W, expert_order(ids, 10)), species_linear(x, W, ids).double()) < 2e-5


def test_graph_replays(device):
    from ictc_o3 import expert_linear, expert_order
    ids, x, W, b, gy = _inputs(700, 5, 64, 96, torch.float32, 10, device)
    args = [t.clone().requires_grad_() for t in (x, W, b)]
    order = expert_order(ids, 5)

    def step():
        y = expert_linear(args[0], args[1], order, args[2])
        return (y, *torch.autograd.grad(y, args, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            args[0].mul_(0.5)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(i, j) for i, j in zip(held, eager)), k


@pytest.mark.parametrize("rows", [0, 1, 63, 64, 65, 1000, 1025, 8191, 16384, 16385, 40000])
@pytest.mark.parametrize("experts", [1, 2, 10, 89, 1023, 1024, 5000])
def test_order(device, rows, experts):
    """The stable order of the ids, those of no expert last."""
    from ictc_o3 import expert_order
    g = torch.Generator().manual_seed(rows + experts)
    ids = torch.randint(-2, experts + 2, (rows,), generator=g)
    if rows > 100:
        ids[:50] = experts - 1
        ids[60] = 2 ** 40
    order = expert_order(ids.to(device), experts)
    key = torch.where((ids >= 0) & (ids < experts), ids, torch.full_like(ids, experts))
    ref = torch.sort(key, stable=True).indices
    assert torch.equal(order.perm[:rows].cpu().long(), ref)
    starts = torch.searchsorted(key[ref], torch.arange(experts + 1))
    assert torch.equal(order.offsets.cpu().long(), torch.cat([starts, torch.tensor([rows])]))


@pytest.mark.parametrize("rows", [8571, 8572, 12288, 65537, 262145, 1048577, 4194305])
@pytest.mark.parametrize("experts", [1, 10, 300, 1023])
def test_order_of_many_rows(device, rows, experts):
    """Blocks that each place a part of the rows, whole parts and a last one of one row."""
    from ictc_o3 import expert_order
    ids = torch.randint(-1, experts + 1, (rows,), device=device, generator=torch.Generator(device).manual_seed(rows + experts))
    order = expert_order(ids, experts)
    key = torch.where((ids >= 0) & (ids < experts), ids, torch.full_like(ids, experts))
    placed = order.perm[:rows].long()
    assert torch.equal(torch.bincount(placed, minlength=rows), torch.ones(rows, dtype=torch.int64, device=device))
    assert (torch.diff(key[placed] * rows + placed) > 0).all()   # by expert, then by row
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=device), torch.bincount(key, minlength=experts + 1).cumsum(0)])
    assert torch.equal(order.offsets.long(), starts)


def test_refusals(device):
    from ictc_o3 import expert_linear, expert_order
    ids = torch.zeros(6, dtype=torch.int64, device=device)
    order = expert_order(ids, 2)
    x, W, b = torch.ones(6, 4, device=device), torch.ones(2, 5, 4, device=device), torch.ones(2, 5, device=device)
    for bad in (dict(x=x.double()), dict(x=x.bfloat16()), dict(x=x[:5]), dict(x=x[:, :3]), dict(W=W[:1]), dict(W=W[0]),
                dict(b=b[:, :4]), dict(b=b.half()), dict(W=W.cpu()), dict(W=W[:, :0])):
        a = dict(x=x, W=W, b=b)
        a.update(bad)
        with pytest.raises(ValueError):
            expert_linear(a["x"], a["W"], order, a["b"])
    with pytest.raises(TypeError):
        expert_linear(x, W, ids)
    for bad in ((ids.int(), 2), (ids.view(2, 3), 2), (ids, 0), (ids, 70000), (ids, 2.0), (ids.cpu(), 2)):
        with pytest.raises(ValueError):
            expert_order(*bad)


@pytest.mark.parametrize("dtype,K,M", [(torch.bfloat16, 1000, 72), (torch.float16, 17, 1001)])
def test_offsets_past_32_bits(device, dtype, K, M):
    """Rows or outputs of more than 2^31 elements: the first and last rows, and their gradients alone."""
    from ictc_o3 import expert_linear, expert_order
    N, E = 2200000, 5
    g = torch.Generator(device).manual_seed(1)
    x = torch.randn(N, K, device=device, dtype=dtype, generator=g).requires_grad_()
    ids = torch.randint(0, E, (N,), device=device, generator=g)
    W = (torch.randn(E, M, K, device=device, generator=g) / math.sqrt(K)).to(dtype).requires_grad_()
    y = expert_linear(x, W, expert_order(ids, E))
    ends = torch.cat([torch.arange(0, 200, device=device), torch.arange(N - 200, N, device=device)])
    gy = torch.zeros(N, M, device=device, dtype=dtype)
    gy[ends] = torch.randn(400, M, device=device, generator=g).to(dtype)
    gx, gW = torch.autograd.grad(y, (x, W), gy)
    few = [t.detach().double().requires_grad_() for t in (x[ends], W)]
    Y = _formula(*few, None, ids[ends])
    _check((y[ends], gx[ends], gW), (Y, *torch.autograd.grad(Y, few, gy[ends].double())), ("y", "gx", "gW"))
    assert gx[200:400].abs().max() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K,M", [(40, 300, 64), (1000, 128, 72), (1000, 65, 33), (900, 5, 7)])
def test_non_finite_rows_stay_alone(device, rows, K, M, dtype):
    """Infinities and NaN in some rows change neither other rows' results nor other experts' gradients."""
    ids, x, W, b, gy = _inputs(rows, 4, K, M, dtype, 21, device)
    bad = x.clone()
    bad[5, K // 2], bad[9, 0], bad[rows // 2], bad[rows - 1] = float("inf"), float("-inf"), float("nan"), float("nan")
    ids[5], ids[9], ids[rows // 2] = 0, 0, 0
    _, y0, clean = _run(ids, x, W, b, gy)
    _, y1, got = _run(ids, bad, W, b, gy)
    others = torch.ones(rows, dtype=torch.bool, device=device)
    others[[5, 9, rows // 2]] = False          # (the last row belongs to no expert)
    assert torch.equal(y1[others], y0[others]) and not torch.isfinite(y1[~others]).all(1).any()
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert torch.equal(got[1][1:], clean[1][1:]) and not torch.isfinite(got[1][0]).all()


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("K,M", [(264, 504), (504, 264), (256, 1000)])
def test_many_rows_and_columns(device, dtype, K, M):
    """Rows and columns enough for the largest tiles, straight and transposed, the last ones part full."""
    data = _inputs(50021, 3, K, M, dtype, K, device)
    _, y, got = _run(*data)
    _, Y, ref = _reference(*data)
    _check((y, *got), (Y, *ref), ("y", "gx", "gW", "gb"))


def test_the_same_without_a_graph(device):
    from ictc_o3 import expert_linear, expert_order
    ids, x, W, b, _ = _inputs(60, 3, 40, 24, torch.float32, 6, device)
    order = expert_order(ids, 3)
    plain, kept = expert_linear(x, W, order, b), expert_linear(x, W, order, b.clone().requires_grad_())
    with torch.no_grad():
        off = expert_linear(x.clone().requires_grad_(), W, order, b)
    with torch.inference_mode():
        inference = expert_linear(x, W, expert_order(ids, 3), b)
    assert kept.requires_grad and not plain.requires_grad and not off.requires_grad
    assert all(torch.equal(t, kept) for t in (plain, off, inference))


@pytest.mark.parametrize("rows,K,M", [(50021, 264, 504), (50021, 504, 264), (50021, 263, 501), (50021, 501, 263), (70000, 256, 256), (70001, 255, 257)])
def test_many_rows_and_columns_in_fp32(device, rows, K, M):
    """The largest FP32 tiles of rows, adjoint and weights' gradient, aligned and not, the last ones part full."""
    data = _inputs(rows, 3, K, M, torch.float32, K, device)
    _, y, got = _run(*data)
    _, Y, ref = _reference(*data)
    _check((y, *got), (Y, *ref), ("y", "gx", "gW", "gb"))
    _, y2, again = _run(*data)
    assert torch.equal(y, y2) and all(torch.equal(i, j) for i, j in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("K,M", [(201, 333), (333, 201), (511, 131)])
def test_odd_rows_of_many_steps(device, dtype, K, M):
    """Rows that are not 16-byte aligned, reductions of several steps straight and transposed."""
    data = _inputs(40000, 4, K, M, dtype, K, device)
    _, y, got = _run(*data)
    _, Y, ref = _reference(*data)
    _check((y, *got), (Y, *ref), ("y", "gx", "gW", "gb"))


FORMS = [(16, 8, 1024, 256), (900, 2, 3, 5), (900, 3, 64, 96), (3000, 3, 128, 100), (3000, 3, 129, 101), (70000, 3, 256, 256),
         (70001, 3, 255, 257)]


@pytest.mark.parametrize("rows,experts,K,M", FORMS)
def test_fp32_values_of_any_size(device, rows, experts, K, M):
    """Values from 2^-60 to 2^60 whose products are of one size, within a row and from row to row.  FP32 operands are split
    into three parts whatever their exponents, and powers of two change no other rounding, so once they are taken out
    of the results the bound is that of values of one size."""
    ids, x, W, b, gy = _inputs(rows, experts, K, M, torch.float32, rows, device)
    g = torch.Generator().manual_seed(4)
    s = torch.exp2(torch.randint(-60, 61, (K,), generator=g).float()).to(device)
    t = torch.exp2(torch.randint(-60, 61, (M,), generator=g).float()).to(device)
    for first in ("inputs", "outputs"):        # sizes that cancel in y and gW's rows, then in gx
        if first == "inputs":
            data = (ids, x * s, W / s, b, gy)
        else:
            data = (ids, x, W / t[:, None], b / t, gy * t)
        _, y, got = _run(*data)
        _, Y, ref = _reference(*data)
        gx, gW, gb = got
        GX, GW, GB = ref
        if first == "inputs":
            pairs = ((y, Y), (gx * s, GX * s.double()), (gW / s, GW / s.double()), (gb, GB))
        else:
            pairs = ((y * t, Y * t.double()), (gx, GX), (gW / t[:, None], GW / t.double()[:, None]), (gb / t, GB / t.double()))
        _check([p[0] for p in pairs], [p[1] for p in pairs], ("y", "gx", "gW", "gb"))
    r = torch.exp2(torch.randint(-60, 61, (rows,), generator=g).float()).to(device)[:, None]    # cancel in gW
    data = (ids, x * r, W, torch.zeros_like(b), gy / r)
    _, y, got = _run(*data)
    _, Y, ref = _reference(*data)
    _check((y / r, got[0] * r, got[1]), (Y / r.double(), ref[0] * r.double(), ref[1]), ("y", "gx", "gW"))


def test_gradients_of_gradients_in_bfloat16(device):
    """Of several first gradients at once: each second one is a single product, rounded once."""
    data = _inputs(300, 4, 40, 72, torch.bfloat16, 2, device)
    args, y, first = _run(*data, create=True)
    Args, Y, First = _reference(*data)
    g = torch.Generator().manual_seed(3)
    v = [torch.randn(t.shape, generator=g).to(torch.bfloat16).to(device) for t in first]
    got = torch.autograd.grad(first[:2], args[:2], v[:2], create_graph=True)
    ref = torch.autograd.grad(First[:2], Args[:2], [t.double() for t in v[:2]], create_graph=True)
    _check(got, ref, ("by x", "by W"))


def test_fp32_values_near_the_smallest(device):
    """A value's third part ends at bfloat16's last bit, 2^-133, so a value is off by up to 2^-134: of K = 64 terms, a
    result by sum |w| 2^-134 at most; and by the bound of any result.  Results are kept large by the weights."""
    from ictc_o3 import expert_linear, expert_order
    for rows in (16, 3000, 70000):
        ids, x, W, _, _ = _inputs(rows, 2, 64, 256, torch.float32, rows, device, bad=False)
        order = expert_order(ids, 2)
        for e in (-100, -110, -118, -126):
            small, large = x * 2.0 ** e, W * 2.0 ** 90
            Y = _formula(small.double(), large.double(), None, ids)
            off = (expert_linear(small, large, order).double() - Y).abs().max()
            lost = large.double().abs().sum(2).max() * 2.0 ** -134 if e < -110 else 0.0
            assert off < 2e-5 * Y.abs().max() + lost, (rows, e)
