"""Traces of the dense layers' operators are refused: a trace would keep the allocation of a result and not the kernel
that writes it.  (No GPU work is reached: the refusal comes before the operands are looked at.)"""
import os

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

TRACERS = [lambda f: torch.jit.trace(f, torch.ones(2, 4), check_trace=False), lambda f: make_fx(f)(torch.ones(2, 4)),
           lambda f: make_fx(f, tracing_mode="fake")(torch.ones(2, 4))]


def _calls():
    import ictc_o3
    from ictc_o3 import _native as nat
    ids, m = torch.zeros(2, dtype=torch.int64), torch.zeros(256)
    return [lambda x: ictc_o3.layer_norm(x),
            lambda x: ictc_o3.expert_order(x.long()[:, 0], 2).perm,
            lambda x: nat.ops().expert_linear(x, torch.ones(1, 4, 4), None, ids, ids, 2),
            lambda x: ictc_o3.adamw_step([x], [x], m, m, step=1, max_norm=1.0),
            lambda x: ictc_o3.adamw_moments(x, x, x, x)]


@pytest.mark.parametrize("call", range(5))
@pytest.mark.parametrize("tracer", range(3))
def test_refused(tracer, call):
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    f = _calls()[call]
    with pytest.raises(ValueError, match="trac"):
        TRACERS[tracer](f)
    with pytest.raises(ValueError) as said:
        f(torch.ones(2, 4))
    assert "trac" not in str(said.value)
