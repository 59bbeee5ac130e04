"""AdamW over many tensors against its formula in float64, its 8-bit moments against codes made by torch, the optimizer
class against torch.optim.AdamW in float64, and refusals.

Bounds: a moment takes at most seven roundings of FP32 (three of them the gradient's factor), a parameter nine, each
2^-24 of a value no larger than the largest term: 9 * 2^-24 = 5.4e-7; the bound is 1e-6 of the largest value, times the
number of steps taken.  A bfloat16 or float16 parameter is rounded once more: 2^-9 or 2^-11, the bounds are twice that.
Codes and scales have to be equal, bit by bit: without a norm bound every operation on the moments is rounded alone.
"""
import copy

import pytest
import torch

from helpers import rel_err

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-6, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [1, 3, 255, 256, 257, 64, 2047, 2048, 2049, 10000, 0, 17]


def _formula(p, g, m, v, step, max_norm=None, *, lr, betas, eps, weight_decay):
    norm = torch.cat([x.flatten() for x in g]).norm() if max_norm is not None else None
    c = min(1.0, max_norm / (float(norm) + 1e-6)) if max_norm is not None else 1.0
    out = []
    for a, b, i, j in zip(p, g, m, v):
        b = b * c
        i = betas[0] * i + (1 - betas[0]) * b
        j = betas[1] * j + (1 - betas[1]) * b * b
        up = i / (1 - betas[0] ** step) / ((j / (1 - betas[1] ** step)).sqrt() + eps)
        out.append((a * (1 - lr * weight_decay) - lr * up, i, j))
    return [list(t) for t in zip(*out)], norm


def _lists(sizes, dtype, seed, device, odd=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for scale in (0.3, 0.02):
        ts = []
        for n in sizes:
            t = (scale * torch.randn(n + 1, generator=g)).to(dtype).to(device)
            ts.append(t[1:] if odd else t[:-1].clone())
        out.append(ts)
    return out


def _segments(flat, starts, sizes):
    return [flat[a:a + n] for a, n in zip(starts, sizes)]


@pytest.mark.parametrize("max_norm", [None, 0.05, 1e6])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_step_against_the_formula(device, dtype, odd, max_norm):
    from ictc_o3 import adamw_segments, adamw_step
    ps, gs = _lists(SIZES, dtype, 1, device, odd)
    starts, total = adamw_segments(SIZES)
    assert starts[:5] == [0, 256, 512, 768, 1024] and total % 256 == 0
    m, v = torch.zeros(total, device=device), torch.zeros(total, device=device)
    for step in (1, 2, 700):
        old = [[t.double() for t in ts] for ts in (ps, gs, _segments(m, starts, SIZES), _segments(v, starts, SIZES))]
        before = [t.clone() for t in gs]
        norm = adamw_step(ps, gs, m, v, step=step, max_norm=max_norm, **HYPER)
        (P, M, V), N = _formula(*old, step, max_norm, **HYPER)
        assert all(torch.equal(a, b) for a, b in zip(gs, before))
        assert (norm is None) == (max_norm is None)
        if norm is not None:
            assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - float(N)) < 1e-6 * float(N)
        for got, ref, tol in ((ps, P, TOL[dtype]), (_segments(m, starts, SIZES), M, 1e-6),
                              (_segments(v, starts, SIZES), V, 1e-6)):
            assert rel_err(torch.cat([t.flatten() for t in got]), torch.cat(ref)) < tol
        filled = torch.zeros(total, dtype=torch.bool, device=device)
        for a, n in zip(starts, SIZES):
            filled[a:a + n] = True
        assert m[~filled].abs().max() == 0 and v[~filled].abs().max() == 0


def test_more_tensors_than_one_launch_takes(device):
    from ictc_o3 import adamw_segments, adamw_step
    sizes = [1 + (i * 97) % 700 for i in range(263)]
    ps, gs = _lists(sizes, torch.float32, 2, device)
    starts, total = adamw_segments(sizes)
    m, v = torch.zeros(total, device=device), torch.zeros(total, device=device)
    old = [[t.double() for t in ts] for ts in (ps, gs, _segments(m, starts, sizes), _segments(v, starts, sizes))]
    norm = adamw_step(ps, gs, m, v, step=1, max_norm=0.1, **HYPER)
    (P, M, V), N = _formula(*old, 1, 0.1, **HYPER)
    assert abs(float(norm) - float(N)) < 1e-6 * float(N)
    assert rel_err(torch.cat(ps), torch.cat(P)) < 1e-6
    assert rel_err(torch.cat(_segments(v, starts, sizes)), torch.cat(V)) < 1e-6


# ---------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------


def _encode(m, v):
    """Codes and scales of FP32 moments [blocks, 256] by torch on the CPU."""
    m, v = m.cpu().view(-1, 256), v.cpu().view(-1, 256)
    em = (torch.frexp(m.abs().amax(1)).exponent - 8).clamp(-126, 126)
    sm = torch.tensor([2.0 ** int(e) for e in em])
    cm = (m.double() / sm.double()[:, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    scale, codes = [], []
    for row in v.double():
        top = float(row.max())
        mant, e = torch.frexp(torch.tensor(top, dtype=torch.float64))
        e = int(e) - 1 + (1 if float(mant) >= 31.0 / 32.0 else 0)      # the maximum rounds up to the next power of two
        e = max(-126, min(126, e)) if top > 0 else -126
        y = row / 2.0 ** e
        mant, k = torch.frexp(y)
        q = torch.round(mant * 16)                                     # 8 .. 16, ties to even
        k = k - 1 + (q == 16)
        q = torch.where(q == 16, torch.full_like(q, 8.0), q)
        c = ((k + 31) * 8 + q - 8).clamp(1, 255)
        codes.append(torch.where(row > 0, c, torch.zeros_like(c)).to(torch.uint8))
        scale.append(2.0 ** e)
    return cm.view(-1), sm, torch.stack(codes).view(-1), torch.tensor(scale)


def _values(c, s):
    x = c.double()
    return torch.where(x > 0, (1 + x % 8 / 8) * 2.0 ** (torch.div(x, 8, rounding_mode="floor") - 31), 0 * x) \
        * s.double().repeat_interleave(256)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_of_8_bit_moments(device, dtype):
    from ictc_o3 import adamw_moments, adamw_segments, adamw_step
    sizes = [300, 256, 5, 2304, 1, 700]
    ps, gs = _lists(sizes, dtype, 3, device)
    gs[1].mul_(1e6)
    gs[2].zero_()
    gs[3] *= torch.exp2(-torch.arange(2304, device=device) / 64).to(dtype)     # 36 binades within nine blocks
    gs[5][::3] = 0
    starts, total = adamw_segments(sizes)
    m8 = torch.zeros(total, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    v8 = torch.zeros(total, dtype=torch.uint8, device=device)
    sm, sv = torch.ones(total // 256, device=device), torch.ones(total // 256, device=device)
    m, v = torch.zeros(total), torch.zeros(total)
    b1, b2 = HYPER["betas"]
    f = torch.float32
    for step in range(1, 5):
        old_p = torch.cat([p.double().flatten() for p in ps]).cpu()
        adamw_step(ps, gs, m8, v8, step=step, exp_avg_scale=sm, exp_avg_sq_scale=sv, **HYPER)
        for a, n, g in zip(starts, sizes, gs):
            g = g.cpu().float()
            m[a:a + n] = m[a:a + n] * torch.tensor(b1, dtype=f) + g * torch.tensor(1 - b1, dtype=f)
            v[a:a + n] = v[a:a + n] * torch.tensor(b2, dtype=f) + g * g * torch.tensor(1 - b2, dtype=f)
        new = []
        for a, n in zip(starts, sizes):
            up = m[a:a + n].double() / (1 - b1 ** step) / ((v[a:a + n].double() / (1 - b2 ** step)).sqrt() + 1e-8)
            new.append(up)
        ref = old_p * (1 - HYPER["lr"] * HYPER["weight_decay"]) - HYPER["lr"] * torch.cat(new)
        assert rel_err(torch.cat([p.flatten() for p in ps]), ref) < TOL[dtype]
        cm, cs, cv, vs = _encode(m, v)
        assert torch.equal(m8.view(torch.uint8).cpu(), cm) and torch.equal(v8.cpu(), cv)
        live = m.view(-1, 256).abs().amax(1) > 0
        assert torch.equal(sm.cpu()[live], cs[live]) and torch.equal(sv.cpu()[live], vs[live])
        assert ((v8.cpu() > 0) == (v > 0)).all()                               # nothing small became zero
        for kind in (torch.float32, torch.bfloat16):
            dm, dv = adamw_moments(m8, v8, sm, sv, dtype=kind)
            m = (cm.view(torch.float8_e4m3fn).double() * cs.double().repeat_interleave(256)).float()
            assert torch.equal(dm.cpu().float()[live.repeat_interleave(256)], m[live.repeat_interleave(256)])
            v = _values(cv, vs).float()
            assert torch.equal(dv.cpu().float(), v)


def test_8_bit_moments_of_extreme_gradients(device):
    """Values near both ends of FP32: scales are held to 2^-126 .. 2^126 and nothing becomes NaN."""
    from ictc_o3 import adamw_moments, adamw_step
    for size in (1e-38, 1e-25, 1e-12, 1e12, 1.5e19):
        g = torch.full((256,), size, device=device)
        p = torch.zeros(256, device=device)
        m8 = torch.zeros(256, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        v8 = torch.zeros(256, dtype=torch.uint8, device=device)
        sm, sv = torch.ones(1, device=device), torch.ones(1, device=device)
        adamw_step([p], [g], m8, v8, step=1, exp_avg_scale=sm, exp_avg_sq_scale=sv, **{**HYPER, "eps": 0.0 if size > 1e-15 else 1e-8})
        m, v = adamw_moments(m8, v8, sm, sv)
        assert torch.isfinite(p).all() and torch.isfinite(m).all() and torch.isfinite(v).all()
        assert abs(float(m[0]) / (0.1 * size) - 1) < 1 / 16 or size < 1e-36
        if size * size > 1e-35:
            assert abs(float(v[0]) / (0.01 * size * size) - 1) < 1 / 16


@pytest.mark.parametrize("bits", [32, 8])
def test_nan_and_infinity_reach_only_their_own(device, bits):
    from ictc_o3 import AdamW
    for bad in (float("nan"), float("inf")):
        ps = [torch.nn.Parameter(torch.ones(n, device=device)) for n in (700, 40)]
        opt = AdamW(ps, state_bits=bits)
        for p in ps:
            p.grad = torch.full_like(p, 0.5)
        ps[0].grad[300] = bad
        opt.step()
        fine = torch.ones(700, dtype=torch.bool, device=device)
        fine[300] = False
        assert torch.isfinite(ps[0][fine]).all() and not torch.isfinite(ps[0][300]) and torch.isfinite(ps[1]).all()
        ps[0].grad[300] = 0.5
        opt.step()
        if bits == 8:     # the block's scale is lost with it: loud, and the other blocks go on
            fine[256:512] = False
        assert torch.isfinite(ps[0][fine]).all() and not torch.isfinite(ps[0][300])
        assert torch.isfinite(ps[1]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[1], [0, 5, 0], [2048 * 8], [2048 * 8 + 1], [2048] * 8, [300] * 9, [1] * 121, [2049, 7, 6000]])
def test_norms_of_few_elements(device, dtype, counts):
    """Squares and eight of them are added in FP32, under five units of 2^-24 of the norm, and the norm is rounded."""
    from ictc_o3 import AdamW
    g = torch.Generator().manual_seed(sum(counts))
    ps = [torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=device)) for n in counts]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).to(dtype).to(device)
    opt = AdamW(ps, max_norm=0.5)
    opt.step()
    ref = torch.cat([p.grad.double() for p in ps]).norm()
    assert abs(float(opt.grad_norm) - float(ref)) < 1e-6 * float(ref)


def test_a_bound_with_a_non_finite_norm_is_loud(device):
    from ictc_o3 import adamw_step
    p, g = torch.ones(300, device=device), torch.ones(300, device=device)
    g[7] = float("nan")
    m, v = torch.zeros(512, device=device), torch.zeros(512, device=device)
    norm = adamw_step([p], [g], m, v, step=1, max_norm=1.0)
    assert torch.isnan(norm) and torch.isnan(p).all()


def test_offsets_past_32_bits(device):
    """2^31 + 777 bfloat16 parameters with 8-bit moments: elements at both ends, against a small tensor's."""
    from ictc_o3 import adamw_segments, adamw_step
    n = 2 ** 31 + 777
    _, total = adamw_segments([n])

    def state(total):
        return (torch.zeros(total, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                torch.zeros(total, dtype=torch.uint8, device=device), torch.ones(total // 256, device=device),
                torch.ones(total // 256, device=device))

    p = torch.zeros(n, dtype=torch.bfloat16, device=device)
    g = torch.zeros(n, dtype=torch.bfloat16, device=device)
    ends = torch.randn(1000, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(device)
    p[:1000], g[:1000], p[-1000:], g[-1000:] = ends, ends.flip(0), ends, ends.flip(0)
    m, v, sm, sv = state(total)
    norm = adamw_step([p], [g], m, v, step=1, exp_avg_scale=sm, exp_avg_sq_scale=sv, max_norm=1e9, **HYPER)
    small = ends.clone()
    m2, v2, sm2, sv2 = state(1024)
    adamw_step([small], [ends.flip(0)], m2, v2, step=1, exp_avg_scale=sm2, exp_avg_sq_scale=sv2, **HYPER)
    assert torch.equal(p[:1000], small) and torch.equal(p[-1000:], small)
    assert p[1000:2000].abs().max() == 0
    assert abs(float(norm) - 2 ** 0.5 * float(ends.double().norm())) < 1e-5 * float(norm)


# ---------------------------------------------------------------------------
# The optimizer
# ---------------------------------------------------------------------------


def _pair(device, shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    start = [torch.randn(s, generator=g, dtype=torch.float64) for s in shapes]
    return ([torch.nn.Parameter(t.float().to(device)) for t in start],
            [torch.nn.Parameter(t.float().double()) for t in start])


def test_optimizer_against_torch(device):
    """Eight steps with two groups, a learning rate schedule and a parameter that some steps give no gradient."""
    from ictc_o3 import AdamW
    ps, rs = _pair(device, [(7, 5), (300,), (2, 3, 64), (1,), (500,)])
    groups = lambda q: [dict(params=q[:3], weight_decay=0.1), dict(params=q[3:], lr=1e-2)]  # noqa: E731
    opt = AdamW(groups(ps), lr=1e-3, max_norm=0.7)
    ref = torch.optim.AdamW(groups(rs), lr=1e-3, eps=1e-8)
    sched = [torch.optim.lr_scheduler.StepLR(o, 3, 0.5) for o in (opt, ref)]
    gen = torch.Generator().manual_seed(9)
    for k in range(8):
        for i, (p, r) in enumerate(zip(ps, rs)):
            grad = torch.randn(r.shape, generator=gen)
            skip = i == 1 and k in (0, 3)
            p.grad, r.grad = (None, None) if skip else (grad.to(device), grad.double())
        norm = torch.nn.utils.clip_grad_norm_([r for r in rs if r.grad is not None], 0.7)
        opt.step()
        ref.step()
        for s in sched:
            s.step()
        assert abs(float(opt.grad_norm) - float(norm)) < 1e-6 * float(norm)
    for p, r in zip(ps, rs):
        assert rel_err(p, r) < 8e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_saved_state_continues_bit_by_bit(device, bits, dtype, tmp_path):
    from ictc_o3 import AdamW
    ps = [torch.nn.Parameter(p.detach().to(dtype)) for p in _pair(device, [(600,), (33, 9)])[0]]
    opt = AdamW(ps, lr=1e-2, state_bits=bits)
    gen = torch.Generator().manual_seed(4)
    grads = [[torch.randn(p.shape, generator=gen).to(dtype).to(device) for p in ps] for _ in range(6)]

    def steps(opt, ps, which):
        for k in which:
            for p, g in zip(ps, grads[k]):
                p.grad = g
            opt.step()

    steps(opt, ps, range(3))
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    for how in ("file", "copy"):
        qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        if how == "file":
            other = AdamW(qs, lr=1.0, state_bits=bits)
            other.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
            assert other.param_groups[0]["lr"] == 1e-2
        else:
            other = copy.deepcopy(opt)
            qs = other.param_groups[0]["params"]
        keep = [p.detach().clone() for p in ps]
        state = copy.deepcopy(opt.state_dict())
        steps(other, qs, range(3, 6))
        assert all(torch.equal(a, b) for a, b in zip(keep, ps))                 # the first one was left alone
        mine = AdamW([torch.nn.Parameter(t) for t in keep], lr=1e-2, state_bits=bits)
        mine.load_state_dict(state)
        again = mine.param_groups[0]["params"]
        steps(mine, again, range(3, 6))
        assert all(torch.equal(a, b) for a, b in zip(again, qs)), how
    wrong = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=40 - bits)
    state = opt.state_dict()
    state["param_groups"][0]["state_bits"] = 40 - bits
    wrong.load_state_dict(state)
    for p, g in zip(wrong.param_groups[0]["params"], grads[0]):
        p.grad = g
    with pytest.raises(ValueError, match="state"):
        wrong.step()


def test_8_bits_fit_as_well_as_32(device):
    """A least-squares fit: both kinds of moments come down to the same loss within a tenth."""
    from ictc_o3 import AdamW
    g = torch.Generator().manual_seed(0)
    A = torch.randn(512, 300, generator=g).to(device)
    y = A @ torch.randn(300, 4, generator=g).to(device) + 0.5 * torch.randn(512, 4, generator=g).to(device)
    loss = {}
    for bits in (32, 8):
        w = torch.nn.Parameter(torch.zeros(300, 4, device=device))
        opt = AdamW([w], lr=2e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(400):
            opt.zero_grad()
            out = (A @ w - y).square().mean()
            out.backward()
            opt.step()
        loss[bits] = float(out)
    assert loss[8] < 1.1 * loss[32] < 0.2


def test_a_step_outdates_what_was_read_of_a_parameter(device):
    """Cached weight copies and saved graph inputs go by a tensor's version: a step has to change it."""
    from ictc_o3 import AdamW
    p = torch.nn.Parameter(torch.ones(64, 64, device=device))
    x = torch.ones(2, 64, device=device, requires_grad=True)
    y = (x @ p).sum()
    before = p._version
    p.grad = torch.ones_like(p)
    AdamW([p]).step()
    assert p._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_gradients_of_any_layout_and_other_streams(device):
    from ictc_o3 import AdamW
    ps = [torch.nn.Parameter(torch.ones(40, 30, device=device)) for _ in range(2)]
    grad = torch.randn(30, 40, device=device)
    ps[0].grad, ps[1].grad = grad.t(), grad.t().contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt = AdamW(ps)
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ps[0], ps[1]) and not torch.equal(ps[0], torch.ones_like(ps[0]))


def test_refusals(device):
    from ictc_o3 import adamw_step
    p, g = torch.ones(300, device=device), torch.ones(300, device=device)
    m, v = torch.zeros(512, device=device), torch.zeros(512, device=device)
    bad = [dict(params=[p], grads=[]), dict(grads=[g.double()]), dict(grads=[g[:299]]), dict(params=[p.cpu()]),
           dict(params=[torch.ones(600, device=device)[::2]]), dict(exp_avg=m[:256]), dict(exp_avg=m[:256], exp_avg_sq=v[:256]),
           dict(exp_avg=m.double()), dict(step=0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(lr=float("nan")),
           dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(exp_avg_scale=torch.ones(2, device=device))]
    for change in bad:
        args = dict(params=[p], grads=[g], exp_avg=m, exp_avg_sq=v, step=1)
        args.update(change)
        with pytest.raises(ValueError):
            adamw_step(**args)
    assert torch.equal(p, torch.ones_like(p))
    assert adamw_step([], [], m, v, step=1) is None


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_join_leave_and_move(device, bits):
    """A group's list of parameters may change between steps: each keeps its own moments and count of steps, as with
    torch.optim.AdamW.  (8 bits against a run in which every parameter has an optimizer of its own.)"""
    from ictc_o3 import AdamW
    ps, rs = _pair(device, [(300,), (5,), (300,), (20, 30)])
    hyper = dict(lr=1e-2, weight_decay=0.05)
    opt = AdamW(ps[:3], state_bits=bits, **hyper)
    if bits == 32:
        refs = [torch.optim.AdamW([r], eps=1e-8, **hyper) for r in rs]
    else:
        rs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        refs = [AdamW([r], state_bits=bits, **hyper) for r in rs]
    gen = torch.Generator().manual_seed(2)
    group = opt.param_groups[0]
    for members in ([0, 1, 2], [0, 1, 2, 3], [1, 2, 3], [3, 2, 1], [2], [0, 2, 1, 3]):
        group["params"][:] = [ps[i] for i in members]
        for _ in range(2):
            for p in ps:
                p.grad = None
            for i in members:
                grad = torch.randn(rs[i].shape, generator=gen)
                ps[i].grad, rs[i].grad = grad.to(device), grad.to(rs[i])
            opt.step()
            for i in members:
                refs[i].step()
        for p, r in zip(ps, rs):
            assert torch.equal(p, r) if bits == 8 else rel_err(p, r) < 12e-6
        if bits == 32:
            for i in members:
                m = opt.state[ps[i]]["exp_avg"][:ps[i].numel()]
                assert rel_err(m, refs[i].state[rs[i]]["exp_avg"].flatten()) < 12e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e25, 1e19, 1e-19, 1e-25, 1e-36])
@pytest.mark.parametrize("counts", [[700], [3000, 5, 20000, 9000]])
def test_norms_whose_squares_leave_the_range(device, dtype, size, counts):
    from ictc_o3 import adamw_segments, adamw_step
    ps, gs = _lists(counts, dtype, 3, device)
    for k, g in enumerate(gs):
        g.mul_(size)
        if k == 1:
            g.mul_(1e-3)
    starts, total = adamw_segments(counts)
    m, v = torch.zeros(total, device=device), torch.zeros(total, device=device)
    old = [[t.double() for t in ts] for ts in (ps, gs, _segments(m, starts, counts), _segments(v, starts, counts))]
    norm = adamw_step(ps, gs, m, v, step=1, max_norm=0.5, **HYPER)
    (P, _, _), N = _formula(*old, 1, 0.5, **HYPER)
    assert abs(float(norm) - float(N)) < 1e-6 * float(N)
    assert rel_err(torch.cat(ps), torch.cat(P)) < TOL[dtype]


def test_a_norm_beyond_the_type_still_scales(device):
    """Every gradient is finite and their norm is past FP32: it is reported as infinite, and the step is the bound's.
    The factor, 2e-41, has 14 bits, and the first step hardly depends on it; the bound is 1e-4."""
    from ictc_o3 import adamw_step
    g = 3e38 * torch.sign(torch.randn(16384, generator=torch.Generator().manual_seed(0))).to(device)
    p, m, v = torch.zeros(16384, device=device), torch.zeros(16384, device=device), torch.zeros(16384, device=device)
    norm = adamw_step([p], [g], m, v, step=1, max_norm=1.0, **HYPER)
    assert torch.isinf(norm)
    assert rel_err(p, -HYPER["lr"] * torch.sign(g).double()) < 1e-4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_of_several_large_tensors(device, dtype):
    from ictc_o3 import adamw_step
    counts = [3000001, 2500000, 7, 4100003, 300, 6000000, 2048, 5000011]
    gen = torch.Generator(device).manual_seed(1)
    gs = [(torch.randn(n, device=device, generator=gen) * (1 + i)).to(dtype) for i, n in enumerate(counts)]
    ps = [torch.zeros_like(g) for g in gs]
    total = sum(-(-n // 256) * 256 for n in counts)
    m, v = torch.zeros(total, device=device), torch.zeros(total, device=device)
    norm = adamw_step(ps, gs, m, v, step=1, max_norm=1.0, **HYPER)
    ref = sum(g.double().square().sum() for g in gs).sqrt()
    assert abs(float(norm) - float(ref)) < 1e-6 * float(ref)


def test_a_bound_does_not_let_a_bad_call_pass(device):
    from ictc_o3 import adamw_step
    p, g = torch.ones(300, device=device), torch.ones(300, device=device)
    m, v = torch.zeros(512, device=device), torch.zeros(512, device=device)
    for bad in (dict(params=[p]), dict(step=0), dict(betas=(1.0, 0.9)), dict(lr=float("nan"))):
        for bound in (None, 1.0):
            with pytest.raises(ValueError):
                adamw_step(**{**dict(params=[], grads=[], exp_avg=m, exp_avg_sq=v, step=1, max_norm=bound), **bad})
    norm = adamw_step([], [], m, v, step=1, max_norm=1.0)
    assert norm.shape == () and float(norm) == 0


def test_a_refused_step_changes_nothing(device):
    from ictc_o3 import AdamW
    ps, rs = _pair(device, [(300,), (40, 30), (77,)])
    hyper = dict(lr=1e-2, weight_decay=0.05)
    groups = lambda q: [dict(params=q[:1]), dict(params=q[1:])]  # noqa: E731
    for bound in (None, 1e9):
        opt = AdamW(groups(ps), max_norm=bound, **hyper)
        gen = torch.Generator().manual_seed(5)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).to(device)
        opt.step()
        state = lambda: copy.deepcopy([[p.detach() for p in ps],  # noqa: E731
                                       [[opt.state[p][k] for k in ("step", "exp_avg", "exp_avg_sq")] for p in ps]])
        before = state()

        def unchanged():
            flat = lambda s: [x for part in s for x in (part if isinstance(part[0], torch.Tensor) else sum(part, []))]  # noqa: E731
            return all(torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b
                       for a, b in zip(flat(before), flat(state())))
        group = opt.param_groups[1]
        for name, bad in (("lr", float("nan")), ("betas", (0.9, 1.0)), ("eps", -1.0), ("weight_decay", float("inf"))):
            good, group[name] = group[name], bad
            with pytest.raises(ValueError):
                opt.step()
            group[name] = good
            assert unchanged(), name
        good = ps[1].data
        ps[1].data, ps[1].grad = good.t().contiguous().t(), ps[1].grad
        with pytest.raises(ValueError, match="contiguous"):
            opt.step()
        assert unchanged()
        ps[1].data = good
        opt.step()
        assert [opt.state[p]["step"] for p in ps] == [2, 2, 2]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("bound", [None, 0.5])
def test_parameters_of_several_types(device, bits, split, bound):
    """FP32, bfloat16 and FP16 in one group or in a group each, one norm over all gradients."""
    from ictc_o3 import AdamW
    types = [torch.float32, torch.bfloat16, torch.float32, torch.float16, torch.bfloat16]
    gen = torch.Generator().manual_seed(7)
    ps = [torch.nn.Parameter(torch.randn(200 + 77 * i, generator=gen).to(t).to(device)) for i, t in enumerate(types)]
    gs = [torch.randn(p.shape, generator=gen).to(p.dtype).to(device) for p in ps]
    groups = [dict(params=[p for p in ps if p.dtype == t]) for t in (torch.bfloat16, torch.float32, torch.float16)]
    opt = AdamW(groups if split else ps, max_norm=bound, state_bits=bits, **HYPER)
    zero = [torch.zeros(p.shape, dtype=torch.float64, device=device) for p in ps]
    (P, _, _), N = _formula([p.detach().double() for p in ps], [g.double() for g in gs], zero, zero, 1, bound, **HYPER)
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    if bound is not None:
        assert opt.grad_norm.dtype == torch.float32 and opt.grad_norm.shape == ()
        assert abs(float(opt.grad_norm) - float(N)) < 1e-6 * float(N)
    for p, r in zip(ps, P):
        assert rel_err(p, r) < TOL[p.dtype]


def test_a_common_norm_of_several_types(device):
    """No bound reached, a bound with one gradient NaN, and norms at both ends of FP32."""
    from ictc_o3 import AdamW
    for size in (1e-30, 1.0, 1e25, float("nan")):
        ps = [torch.nn.Parameter(torch.ones(300, device=device)),
              torch.nn.Parameter(torch.ones(200, device=device, dtype=torch.bfloat16))]
        ps[0].grad = torch.full((300,), size, device=device)
        ps[1].grad = torch.full((200,), 2 * size if size == size else 1.0, device=device, dtype=torch.bfloat16)
        opt = AdamW(ps, max_norm=1e3, **HYPER)
        opt.step()
        if size == size:
            ref = torch.cat([p.grad.double() for p in ps]).norm()
            assert abs(float(opt.grad_norm) - float(ref)) < 1e-6 * float(ref)
            assert all(torch.isfinite(p).all() for p in ps)
        else:
            assert torch.isnan(opt.grad_norm) and all(torch.isnan(p).all() for p in ps)


def test_a_captured_step_is_refused(device):
    """A graph would replay one step's count and rate for ever."""
    from ictc_o3 import AdamW
    p = torch.nn.Parameter(torch.ones(300, device=device))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], max_norm=1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    held = torch.zeros(4, device=device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.add_(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()
    assert opt.state[p]["step"] == 1


def test_codes_of_8_bit_moments_in_half(device):
    """FP16 parameters and gradients: codes and scales bit by bit, as of the other types."""
    from ictc_o3 import adamw_segments, adamw_step
    sizes = [300, 256, 5, 2304, 1, 700]
    ps, gs = _lists(sizes, torch.float16, 3, device)
    gs[1].mul_(1e3)
    gs[2].zero_()
    gs[3] *= torch.exp2(-torch.arange(2304, device=device) / 256).half()
    gs[5][::3] = 0
    starts, total = adamw_segments(sizes)
    m8 = torch.zeros(total, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    v8 = torch.zeros(total, dtype=torch.uint8, device=device)
    sm, sv = torch.ones(total // 256, device=device), torch.ones(total // 256, device=device)
    m, v = torch.zeros(total), torch.zeros(total)
    c = [torch.tensor(x, dtype=torch.float32) for x in (HYPER["betas"][0], 1 - HYPER["betas"][0],
                                                        HYPER["betas"][1], 1 - HYPER["betas"][1])]
    old = [p.double() for p in ps]
    adamw_step(ps, gs, m8, v8, step=1, exp_avg_scale=sm, exp_avg_sq_scale=sv, **HYPER)
    for a, n, g in zip(starts, sizes, gs):
        g = g.cpu().float()
        m[a:a + n] = m[a:a + n] * c[0] + g * c[1]
        v[a:a + n] = v[a:a + n] * c[2] + g * g * c[3]
    cm, cs, cv, vs = _encode(m, v)
    live = m.view(-1, 256).abs().amax(1) > 0
    assert torch.equal(m8.view(torch.uint8).cpu(), cm) and torch.equal(v8.cpu(), cv)
    assert torch.equal(sm.cpu()[live], cs[live]) and torch.equal(sv.cpu()[live], vs[live])
    zero = [torch.zeros_like(p) for p in old]
    (P, _, _), _ = _formula(old, [g.double() for g in gs], zero, zero, 1, None, **HYPER)
    assert rel_err(torch.cat(ps), torch.cat(P)) < TOL[torch.float16]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_cleared_state_starts_anew(device, bits):
    from ictc_o3 import AdamW
    start = [p.detach() for p in _pair(device, [(300,), (20, 30)])[0]]
    gen = torch.Generator().manual_seed(3)
    grads = [[torch.randn(p.shape, generator=gen).to(device) for p in start] for _ in range(3)]

    def steps(opt, ps):
        for gs in grads:
            for p, g in zip(ps, gs):
                p.grad = g
            opt.step()
        return [p.detach().clone() for p in ps]

    ps = [torch.nn.Parameter(p.clone()) for p in start]
    opt = AdamW(ps, lr=1e-2, state_bits=bits)
    first = steps(opt, ps)
    for how in ("clear", "replace"):
        if how == "clear":
            opt.state.clear()
        else:
            opt.state = type(opt.state)(dict)
        with torch.no_grad():
            for p, s in zip(ps, start):
                p.copy_(s)
        assert all(torch.equal(a, b) for a, b in zip(steps(opt, ps), first)), how
        assert [opt.state[p]["step"] for p in ps] == [3, 3]


def test_a_common_norm_beyond_the_type_still_scales(device):
    """As with one type: the factor, 2e-41, has 14 bits, and the first step hardly depends on it; the bound is 1e-4, and
    a bfloat16 parameter's own rounding."""
    from ictc_o3 import AdamW
    signs = torch.sign(torch.randn(16384, generator=torch.Generator().manual_seed(0))).to(device)
    ps = [torch.nn.Parameter(torch.zeros(16384, device=device, dtype=t)) for t in (torch.float32, torch.bfloat16)]
    for p in ps:
        p.grad = (3e38 * signs).to(p.dtype)
    opt = AdamW(ps, max_norm=1.0, **HYPER)
    opt.step()
    assert torch.isinf(opt.grad_norm)
    for p in ps:
        assert rel_err(p, -HYPER["lr"] * signs.double()) < max(1e-4, TOL[p.dtype])
