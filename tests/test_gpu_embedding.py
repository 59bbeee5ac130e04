"""Embedding lookup and its gradient against indexing and sums in float64.

The lookup is one FP32 product rounded once, so it equals that bit for bit.  A sum of m rows in FP32 is off by at most
d 2^-24 of the sum of magnitudes, d the longest chain of additions: no more than m; and no more than 32 rows of a team
(a few more where there are over a million ranges), two runs of each of 256 teams, 1 + ranges / 32 partial sums of a
slice and 32 slices, together under 700 for the sizes here.  Then one product, and one rounding to the type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, entries, width, dtype, device, seed=0, padding=True):
    g = torch.Generator().manual_seed(seed + 7 * rows + entries + width)
    table = torch.randn(entries, width, generator=g).to(dtype).to(device)
    rank = (torch.rand(rows, generator=g) ** 3 * entries).long()       # common and rare entries
    if padding and rows > 2:
        rank[torch.rand(rows, generator=g) < 0.05] = -1
        rank[rows // 2] = entries
    gy = torch.randn(rows, width, generator=g).to(dtype).to(device)
    return table, rank.to(device), gy


def _lookup(table, ids, scale):
    valid = (ids >= 0) & (ids < table.shape[0])
    rows = table.float()[ids.clamp(0, table.shape[0] - 1)] * torch.tensor(scale, dtype=torch.float32)
    return torch.where(valid[..., None], rows, torch.zeros_like(rows)).to(table.dtype)


def _sums(gy, ids, entries, scale):
    valid = (ids >= 0) & (ids < entries)
    g = gy.double()[valid]
    at = ids[valid]
    out = torch.zeros(entries, gy.shape[1], dtype=torch.float64, device=gy.device)
    size, count = torch.zeros_like(out), torch.bincount(at, minlength=entries)
    s = torch.tensor(scale, dtype=torch.float32).double().item()
    return out.index_add(0, at, g) * s, size.index_add(0, at, g.abs()) * abs(s), count


def _check_sums(got, gy, ids, entries, scale):
    ref, size, count = _sums(gy, ids, entries, scale)
    depth = count.clamp(max=700).double()[:, None] + 2
    unit = torch.finfo(gy.dtype).eps / 2
    tiny = torch.finfo(gy.dtype).smallest_normal * unit
    bound = depth * 2.0 ** -24 * size + unit * (ref.abs() + depth * 2.0 ** -24 * size) + tiny
    assert got.dtype == gy.dtype and ((got.double() - ref).abs() <= bound).all()
    assert (got[count == 0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 31, 64, 65, 128, 250, 513, 1021, 2048])
def test_lookup_and_gradient(device, width, dtype):
    from ictc_o3 import embedding, expert_order
    for rows, entries in ((1, 1), (5, 10), (128, 3), (129, 10), (1000, 89), (3001, 2), (2500, 4000), (20011, 10)):
        table, ids, gy = _inputs(rows, entries, width, dtype, device)
        table.requires_grad_()
        y = embedding(table, ids, 2.7)
        assert torch.equal(y, _lookup(table.detach(), ids, 2.7))
        (got,) = torch.autograd.grad(y, table, gy)
        _check_sums(got, gy, ids, entries, 2.7)
        (again,) = torch.autograd.grad(embedding(table, ids, 2.7, order=expert_order(ids, entries)), table, gy)
        assert torch.equal(got, again)          # a fixed order of every sum, whoever sorts


@pytest.mark.parametrize("rows,entries,width,dtype", [(425991, 7921, 64, torch.bfloat16), (131072, 10, 128, torch.float32),
                                                      (60013, 50021, 129, torch.float16), (300000, 1, 8, torch.float32),
                                                      (30000, 140003, 33, torch.float32), (200, 140003, 5, torch.float32),
                                                      (500000, 3, 1, torch.float32)])
def test_many_rows_and_entries(device, rows, entries, width, dtype):
    from ictc_o3 import embedding
    table, ids, gy = _inputs(rows, entries, width, dtype, device)
    table.requires_grad_()
    y = embedding(table, ids, 0.5)
    assert torch.equal(y, _lookup(table.detach(), ids, 0.5))
    got, again = (torch.autograd.grad(embedding(table, ids, 0.5), table, gy)[0] for _ in range(2))
    assert torch.equal(got, again)
    _check_sums(got, gy, ids, entries, 0.5)


def test_runs_that_meet_at_every_border(device):
    """Runs of every length from one to some blocks, one behind another, so that runs begin and end at each place of a
    team, a block and a range; small whole numbers, so sums are exact."""
    from ictc_o3 import embedding
    for width in (4, 60, 300):
        lengths = [k % 97 + 1 for k in range(700)] + [5000, 1, 3000, 2, 129, 128, 127, 512, 513]
        ids = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).to(device)
        table = torch.zeros(len(lengths) + 5, width, device=device, requires_grad=True)
        gy = torch.randint(-8, 9, (ids.shape[0], width), generator=torch.Generator().manual_seed(1)).float().to(device)
        for order in (torch.arange(ids.shape[0], device=device),
                      torch.randperm(ids.shape[0], generator=torch.Generator().manual_seed(2)).to(device)):
            (got,) = torch.autograd.grad(embedding(table, ids[order]), table, gy)
            ref = torch.zeros_like(got).double().index_add(0, ids[order], gy.double())
            assert torch.equal(got.double(), ref)


def test_shapes_strides_and_scalars(device):
    from ictc_o3 import embedding
    table, ids, gy = _inputs(24, 9, 40, torch.float32, device)
    plain = embedding(table, ids)
    assert torch.equal(plain, _lookup(table, ids, 1.0))
    assert torch.equal(embedding(table, ids.view(2, 3, 4)), plain.view(2, 3, 4, 40))
    assert embedding(table, ids[3]).shape == (40,) and torch.equal(embedding(table, ids[3]), plain[3])
    assert torch.equal(embedding(table, ids[::2]), plain[::2])
    assert torch.equal(embedding(table, ids.view(4, 6).t()), plain.view(4, 6, 40).transpose(0, 1))
    assert torch.equal(embedding(table.t().contiguous().t(), ids), plain)           # column-major
    wide = torch.zeros(9, 77, device=device)
    wide[:, 3:43] = table
    assert torch.equal(embedding(wide[:, 3:43], ids), plain)
    assert torch.equal(embedding(table, ids, 0.0), torch.zeros_like(plain))
    wide.requires_grad_()
    for g in (gy, gy.t().contiguous().t(), torch.zeros(24, 91, device=device)[:, 5:45].copy_(gy), gy[:1].expand(24, 40)):
        (got,) = torch.autograd.grad(embedding(wide[:, 3:43], ids, 1.5), wide, g)
        assert (got[:, :3] == 0).all() and (got[:, 43:] == 0).all()
        _check_sums(got[:, 3:43], g, ids, 9, 1.5)


def test_empty(device):
    from ictc_o3 import embedding, expert_order
    table = torch.ones(4, 6, device=device, requires_grad=True)
    none = torch.empty(0, dtype=torch.int64, device=device)
    for order in (None, expert_order(none, 4)):
        y = embedding(table, none, order=order)
        assert y.shape == (0, 6) and (torch.autograd.grad(y, table, torch.empty_like(y))[0] == 0).all()
    y = embedding(table, none.view(3, 0))
    assert y.shape == (3, 0, 6)
    for rows in (3, 300):
        all_padding = torch.full((rows,), -1, dtype=torch.int64, device=device)
        y = embedding(table, all_padding)
        assert (y == 0).all() and (torch.autograd.grad(y, table, torch.ones_like(y))[0] == 0).all()


def test_any_order(device):
    """The map is linear: the gradient's own derivative is the lookup of its cotangent, and so on."""
    from ictc_o3 import embedding
    for rows in (50, 700):
        table, ids, gy = _inputs(rows, 12, 20, torch.float32, device)
        table.requires_grad_()
        gy.requires_grad_()
        (first,) = torch.autograd.grad(embedding(table, ids, 1.25), table, gy, create_graph=True)
        cot = torch.randn_like(table).requires_grad_()
        (second,) = torch.autograd.grad(first, gy, cot, create_graph=True)
        assert torch.equal(second, _lookup(cot.detach(), ids, 1.25))
        (third,) = torch.autograd.grad(second, cot, gy.detach())
        assert torch.equal(third, first)


def test_against_differences(device):
    """The loss is linear in the table but for its square: central differences at step h are exact up to rounding,
    2^-23 of the loss over h = 2^-4 and the gradient's norm, far under the bound 1e-3."""
    from ictc_o3 import embedding
    table, ids, _ = _inputs(300, 7, 16, torch.float32, device)
    table.requires_grad_()
    step = torch.randn_like(table)
    (grad,) = torch.autograd.grad(embedding(table, ids, 3.0).square().sum(), table)
    up, down = (embedding(table.detach() + s * 2.0 ** -4 * step, ids, 3.0).double().square().sum() for s in (1, -1))
    slope = (grad.double() * step.double()).sum()
    assert ((up - down) * 8.0 - slope).abs() < 1e-3 * grad.double().norm() * step.double().norm()


def test_infinities_and_nan_stay_with_their_entry(device):
    from ictc_o3 import embedding
    table, ids, gy = _inputs(400, 6, 33, torch.float32, device, padding=False)
    table[2, 5] = float("inf")
    table[3] = float("nan")
    y = embedding(table, ids)
    assert torch.equal(y.isfinite().all(1), (ids != 2) & (ids != 3))
    gy[(ids == 1).nonzero()[0, 0], 7] = float("nan")
    table = table.detach().requires_grad_()
    (got,) = torch.autograd.grad(embedding(table, ids), table, gy)
    bad = got.isnan()
    assert bad[1, 7] and bad.sum() == 1
    pads = torch.full((200,), -1, dtype=torch.int64, device=device)
    (got,) = torch.autograd.grad(embedding(table, pads), table, torch.full((200, 33), float("nan"), device=device))
    assert (got == 0).all()


def test_streams_and_graph_replays(device):
    from ictc_o3 import embedding, expert_order
    for rows, entries in ((60, 10), (3000, 10), (20000, 700)):
        table, ids, gy = _inputs(rows, entries, 64, torch.float32, device)
        table.requires_grad_()

        def step():
            y = embedding(table, ids, 2.0)
            return y.detach(), *torch.autograd.grad(y, table, gy)

        here = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(here, there))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for k in range(3):
            with torch.no_grad():
                table.add_(0.5)
                gy.mul_(-1.5)
                ids.copy_(ids.roll(11))
            graph.replay()
            eager = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, eager)), k


def test_refusals(device):
    from ictc_o3 import embedding, expert_order
    table, ids, _ = _inputs(20, 5, 8, torch.float32, device)
    order = expert_order(ids, 5)
    for call, match in ((lambda: embedding(table.double(), ids), "float32"),
                        (lambda: embedding(table[0], ids), "shape"),
                        (lambda: embedding(table, ids.int()), "int64"),
                        (lambda: embedding(table, ids.cpu()), "int64"),
                        (lambda: embedding(table[:0], ids), "shape"),
                        (lambda: embedding(table, ids, float("inf")), "finite"),
                        (lambda: embedding(table, ids[:19], order=order), "other ids"),
                        (lambda: embedding(table[:4], ids, order=order), "entries")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError):     # ids changed between the passes
        t = table.clone().requires_grad_()
        y = embedding(t, ids)
        ids.add_(1)
        y.sum().backward()


def test_offsets_past_32_bits(device):
    from ictc_o3 import embedding
    table = torch.zeros(17000003, 128, dtype=torch.bfloat16, device=device)
    ids = torch.cat([torch.arange(50), 17000002 - torch.arange(200)]).to(device)
    g = torch.randn(250, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    table[ids] = g
    table.requires_grad_()
    y = embedding(table, ids)
    assert torch.equal(y, g)
    (got,) = torch.autograd.grad(y, table, g)
    assert torch.equal(got[ids], g) and got[1000:1001000].abs().max() == 0
    del table, got, y
    table = torch.randn(3, 128, device=device, generator=torch.Generator(device).manual_seed(2)).requires_grad_()
    ids = torch.full((17000003,), 1, dtype=torch.int64, device=device)
    ids[-5:] = 2
    y = embedding(table, ids)
    assert torch.equal(y[-6:-4], table[1:].detach()) and torch.equal(y[0], table[1].detach())
    (got,) = torch.autograd.grad(y, table, torch.ones_like(y))
    assert (got[0] == 0).all() and (got[2] == 5).all()
    assert ((got[1].double() - 16999998).abs() <= 16999998 * 700 * 2.0 ** -24).all()


@pytest.mark.parametrize("rows,entries", [(0, 1024), (1, 1023), (1, 1024), (5, 65535), (300, 140003), (16384, 1500),
                                          (20000, 5000), (425991, 7921), (70000, 1048575), (70000, 1048576),
                                          (4300000, 2000), (5000, 33554431), (3, 40000000), (16777216, 10),
                                          (16777217, 10)])
def test_order_of_many_entries(device, rows, entries):
    """The rows' order by id: stable, ids outside last, and where each id begins, whichever passes make it."""
    from ictc_o3 import _native as nat
    g = torch.Generator().manual_seed(rows + entries)
    ids = torch.randint(-2, entries + 3, (rows,), generator=g).to(device)
    if rows > 100:
        ids[rows // 3: rows // 2] = entries // 2        # one id of many
    lib = nat.lib()
    size = lib.ictc_rows_by_id_workspace_bytes(rows, entries)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=device)
    perm = torch.full((max(rows, 1),), -7, dtype=torch.int32, device=device)
    off = torch.full((entries + 2,), -7, dtype=torch.int32, device=device)
    nat.call("ictc_rows_by_id", ids.data_ptr(), rows, entries, perm.data_ptr(), off.data_ptr(), ws.data_ptr(), size,
             torch.cuda.current_stream().cuda_stream)
    key = torch.where((ids >= 0) & (ids < entries), ids, torch.full_like(ids, entries))
    ref = torch.sort(key, stable=True)
    assert torch.equal(perm[:rows].long(), ref.indices)
    counts = torch.bincount(key, minlength=entries + 1)
    assert torch.equal(off.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))


def test_graph_replays_of_very_many_rows(device):
    """More rows than the counted passes take: the general sort, captured and replayed."""
    from ictc_o3 import embedding
    table = torch.randn(50, 2, device=device, requires_grad=True)
    ids = torch.randint(-1, 50, (16777300,), device=device, generator=torch.Generator(device).manual_seed(1))
    gy = torch.ones(16777300, 2, device=device)

    def step():
        return torch.autograd.grad(embedding(table, ids), table, gy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        ids.copy_(ids.roll(1001) if k else ids.flip(0))
        ids[: 1000 * (k + 1)] = k
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(held, eager), k
        ref = torch.bincount(ids[ids >= 0], minlength=50)
        assert ((held[:, 0].double() - ref).abs() <= 700 * 2.0 ** -24 * ref).all()


@pytest.mark.parametrize("rows,entries,kind", [(5, 1024, "near"), (5, 2047, "near"), (300, 3000, "none"), (20000, 4100, "near"),
                                               (129, 1000003, "ends"), (70000, 1000003, "near"), (70000, 1000003, "none"),
                                               (5000, 65535, "spread"), (40000, 33554431, "spread"),
                                               (260, 2 ** 31 - 3, "ends"), (5, 2 ** 31 - 3, "none")])
def test_order_of_ids_side_by_side(device, rows, entries, kind):
    """Ids in one part of a large table, at its ends, or none within it: where each id begins, up to the largest tables."""
    from ictc_o3 import _native as nat
    g = torch.Generator().manual_seed(rows + entries)
    first = entries - 7 if kind == "ends" else entries // 3
    ids = torch.randint(first, min(first + 40, entries + 5), (rows,), generator=g)
    if kind == "ends":
        ids[: rows // 2] = torch.randint(-2, 5, (rows // 2,), generator=g)
    elif kind == "none":
        ids = torch.full((rows,), entries)
    elif kind == "spread":
        ids = torch.randint(0, entries, (rows,), generator=g)
    ids = ids.to(device)
    size = nat.lib().ictc_rows_by_id_workspace_bytes(rows, entries)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=device)
    perm = torch.full((rows,), -7, dtype=torch.int32, device=device)
    off = torch.full((entries + 2,), -7, dtype=torch.int32, device=device)
    nat.call("ictc_rows_by_id", ids.data_ptr(), rows, entries, perm.data_ptr(), off.data_ptr(), ws.data_ptr(), size,
             torch.cuda.current_stream().cuda_stream)
    key = torch.where((ids >= 0) & (ids < entries), ids, torch.full_like(ids, entries))
    ref = torch.sort(key, stable=True)
    assert torch.equal(perm.long(), ref.indices)
    for k in range(0, entries + 2, 1 << 26):
        ks = torch.arange(k, min(entries + 2, k + (1 << 26)), device=device)
        assert torch.equal(off[k:k + (1 << 26)], torch.searchsorted(ref.values, ks, out_int32=True)), k


def test_largest_table(device):
    """A table of 2^31 - 3 entries, the most that are taken: lookup and gradient at its ends."""
    from ictc_o3 import embedding
    entries = 2 ** 31 - 3
    table = torch.zeros(entries, 1, dtype=torch.bfloat16, device=device)
    ids = torch.cat([torch.arange(100), entries - 1 - torch.arange(100), torch.tensor([5, 5, entries, -1, entries - 1])]).to(device)
    inside = (ids >= 0) & (ids < entries)
    gy = torch.randint(-8, 9, (205, 1), generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    table[ids[inside]] = 1.5
    table.requires_grad_()
    y = embedding(table, ids)
    assert torch.equal(y[:, 0], 1.5 * inside)
    (got,) = torch.autograd.grad(y, table, gy)
    ref = torch.zeros(200, dtype=torch.float64, device=device)     # the ends' entries; sums of whole numbers are exact
    ref.index_add_(0, torch.where(ids < 100, ids, ids - entries + 200)[inside], gy[inside, 0].double())
    assert torch.equal(torch.cat([got[:100, 0], got[-100:, 0]]).double(), ref)
    for part in got[100:-100].split(1 << 28):
        assert not part.any()


@pytest.mark.parametrize("rows,entries", [((1 << 21) + 1, 7921), ((12 << 20) + 5, 1000)])
def test_graph_replays_of_the_general_sort(device, rows, entries):
    """Very many rows take the general sort: the order captured and replayed, against the eager one and its definition."""
    from ictc_o3 import expert_order
    ids = torch.randint(-1, entries + 1, (rows,), device=device, generator=torch.Generator(device).manual_seed(1))
    expert_order(ids, entries)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = expert_order(ids, entries)
    for k in range(4):
        ids.copy_(ids.roll(1001) if k else ids.flip(0))
        ids[: 1000 * (k + 1)] = k
        graph.replay()
        eager = expert_order(ids, entries)
        torch.cuda.synchronize()
        assert torch.equal(held.perm, eager.perm) and torch.equal(held.offsets, eager.offsets), k
        key = torch.where((ids >= 0) & (ids < entries), ids, torch.full_like(ids, entries))
        assert torch.equal(held.perm.long(), torch.sort(key, stable=True).indices), k
        counts = torch.bincount(key, minlength=entries + 1)
        assert torch.equal(held.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)])), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [3, 9, 64, 130, 256, 1021])
def test_gradient_of_few_rows_in_a_large_table(device, width, dtype):
    """Up to 128 rows take no order: ids that repeat within and between what a lane holds, single ones, and the table's ends."""
    from ictc_o3 import embedding
    entries = 30011
    for rows in (1, 7, 8, 63, 64, 65, 100, 127, 128):
        g = torch.Generator().manual_seed(rows + width)
        ids = torch.randint(0, entries, (rows,), generator=g)
        ids[::3] = 77
        ids[1::7] = entries - 1
        ids[2::9] = torch.tensor([0, -1, entries, 2 ** 40 + 77, 5]).repeat(26)[: len(ids[2::9])]
        ids = ids.to(device)
        gy = torch.randn(rows, width, generator=g).to(dtype).to(device)
        table = torch.zeros(entries, width, dtype=dtype, device=device, requires_grad=True)
        (got,) = torch.autograd.grad(embedding(table, ids, 1.7), table, gy)
        _check_sums(got, gy, ids, entries, 1.7)


@pytest.mark.parametrize("values", ["alike", "random"])
@pytest.mark.parametrize("rows,width", [(4200001, 256), (4200001, 7)])
def test_sums_of_very_many_rows(device, rows, width, values):
    """Millions of rows of one id.  A sum's additions in FP32: up to 32 rows of a team and 32 teams of a block; its blocks' are
    in FP64, and two roundings follow.  Values alike of 19 bits make every FP32 sum of a block exact, and would lose nearly
    half a unit of a long FP32 sum of blocks in the same direction each time (256 wide 480 units of 2^-24)."""
    from ictc_o3 import embedding
    table = torch.zeros(3, width, device=device, requires_grad=True)
    ids = torch.ones(rows, dtype=torch.int64, device=device)
    ids[:300], ids[-5000:] = 0, 2
    if values == "alike":
        gy = torch.full((rows, width), 1 + 2.0 ** -14 - 2.0 ** -19, device=device)
    else:
        gy = torch.rand(rows, width, device=device, generator=torch.Generator(device).manual_seed(width))
    (got,) = torch.autograd.grad(embedding(table, ids), table, gy)
    parts = gy[:300], gy[300:-5000], gy[-5000:]
    ref = torch.stack([sum(t.double().sum(0) for t in part.split(1 << 18)) for part in parts])
    units = 2 if values == "alike" else 66
    assert ((got.double() - ref).abs() <= units * 2.0 ** -24 * ref).all()
