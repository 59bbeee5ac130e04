"""Refusals of the embedding's entry points (no GPU work is reached)."""
import os

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


def _built():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    return nat


def test_python_refusals():
    nat = _built()
    from ictc_o3 import embedding
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(TypeError):
        embedding([1.0], ids)
    with pytest.raises(TypeError, match="expert_order"):
        embedding(torch.zeros(2, 4), ids, order=(ids, ids))
    with pytest.raises(ValueError, match="device"):
        embedding(torch.zeros(2, 4), ids)
    with pytest.raises(ValueError, match="trac"):
        make_fx(lambda x: nat.ops().embedding(x, ids, 1.0, None, None))(torch.ones(2, 4))
    with pytest.raises(ValueError, match="trac"):
        torch.jit.trace(lambda x: embedding(x, ids), torch.ones(2, 4), check_trace=False)


def test_native_refusals():
    nat = _built()
    size = nat.lib().ictc_embedding_bwd_workspace_bytes
    assert size(0, 100000, 10, 64) > 0 and size(1, 100, 10, 64) == 0 and size(0, 0, 1, 1) == 0
    for bad in ((3, 1, 1, 1), (0, -1, 1, 1), (0, 1, 0, 1), (0, 1, 1, 0), (0, 1, 1, 65537), (0, 2 ** 31, 1, 1),
                (0, 1, 2 ** 31, 1)):
        assert size(*bad) == -1, bad
    needs = nat.lib().ictc_embedding_needs_order
    assert not needs(0) and not needs(128) and needs(129)

    def fwd(dtype=0, table=16, entries=4, width=8, ids=16, rows=2, out=16):
        nat.call("ictc_embedding_fwd", dtype, table, entries, width, ids, rows, 1.0, out, None)

    for bad in (dict(dtype=5), dict(rows=-1), dict(width=0), dict(width=65537), dict(entries=0), dict(table=None),
                dict(ids=None), dict(out=None)):
        with pytest.raises(ValueError):
            fwd(**bad)
    fwd(rows=0, table=None, ids=None, out=None)

    def bwd(dtype=0, grad=16, ldg=8, rows=2000, width=8, ids=16, entries=4, perm=16, off=16, out=16, ws=16, bytes=None):
        bytes = size(0, rows, entries, width) if bytes is None else bytes
        nat.call("ictc_embedding_bwd", dtype, grad, ldg, rows, width, ids, entries, perm, off, 1.0, out, ws, bytes, None)

    assert size(0, 2000, 4, 8) > 0
    for bad in (dict(dtype=-1), dict(ldg=7), dict(grad=None), dict(ids=None), dict(perm=None), dict(off=None),
                dict(out=None), dict(ws=None), dict(ws=18), dict(bytes=4)):
        with pytest.raises(ValueError):
            bwd(**bad)


def test_order_refusals():
    nat = _built()
    size = nat.lib().ictc_rows_by_id_workspace_bytes
    assert size(100, 5) == 0 and size(100000, 200000) > 0
    for bad in ((-1, 5), (5, 0), (2 ** 31, 5), (5, 2 ** 31)):
        assert size(*bad) == -1, bad

    def order(ids=16, rows=100000, entries=200000, perm=16, off=16, ws=16, bytes=1 << 30):
        nat.call("ictc_rows_by_id", ids, rows, entries, perm, off, ws, bytes, None)

    for bad in (dict(ids=None), dict(rows=-1), dict(entries=0), dict(perm=None), dict(off=None), dict(ws=None),
                dict(ws=18), dict(bytes=100)):
        with pytest.raises(ValueError):
            order(**bad)


def test_order_of_very_many_rows():
    """Where the general sort is the faster, the order takes it (and its workspace)."""
    lib = _built().lib()
    for rows, entries, general in ((16777216, 10, False), (16777216, 511, False), (16777217, 10, True),
                                   (12 << 20, 1000, False), ((12 << 20) + 1, 1000, True), (1 << 21, 65535, False),
                                   ((1 << 21) + 1, 65535, True), ((1 << 21) + 1, 1024, True), ((1 << 21) + 1, 40000000, True)):
        assert (lib.ictc_rows_by_id_workspace_bytes(rows, entries) == lib.ictc_csr_workspace_bytes(rows, entries)) == general
        if entries <= 65535:
            assert lib.ictc_expert_order_workspace_bytes(rows, entries) == lib.ictc_rows_by_id_workspace_bytes(rows, entries)


def test_refusals_name_their_own_operator():
    nat = _built()
    for rows, entries in ((100000, 200000), (100000, 1000), (3000000, 200000)):     # passes, one pass, the general sort
        with pytest.raises(ValueError, match="ictc_rows_by_id_workspace_bytes"):
            nat.call("ictc_rows_by_id", 16, rows, entries, 16, 16, None, 0, None)
    for rows, experts in ((100000, 65535), (100000, 1000), (3000000, 65535)):
        with pytest.raises(ValueError, match="ictc_expert_order_workspace_bytes"):
            nat.call("ictc_expert_order", 16, rows, experts, 16, 16, None, 0, None)
