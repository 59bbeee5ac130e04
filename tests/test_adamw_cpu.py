"""Layout and refusals of the AdamW entry points (no GPU work is reached)."""
import os
from array import array

import pytest
import torch


def test_segments():
    from ictc_o3 import adamw_segments
    assert adamw_segments([]) == ([], 0)
    assert adamw_segments([1, 256, 257, 0, 5]) == ([0, 256, 512, 1024, 1024], 1280)


def test_python_refusals():
    from ictc_o3 import AdamW, adamw_moments, adamw_step
    p = torch.ones(4)
    with pytest.raises(ValueError, match="device"):
        adamw_step([p], [p], torch.zeros(256), torch.zeros(256), step=1)
    with pytest.raises(ValueError, match="scales"):
        adamw_moments(torch.zeros(256), torch.zeros(256), None, None)
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(max_norm=-2.0),
                dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(p.clone())], **bad)


def test_native_refusals():
    from ictc_o3 import _native as nat
    if not os.path.exists(nat.library_path()):
        pytest.skip("library not built")
    one, n = array("q", [16]), array("q", [300])
    at = lambda a: a.buffer_info()[0]  # noqa: E731

    def step(dtype=0, bits=32, tensors=1, counts=n, starts=None, m=16, state=512, lr=1e-3, b1=0.9, b2=0.9, eps=1e-8,
             step=1, params=one):
        nat.call("ictc_adamw_step", dtype, bits, tensors, at(params), at(params), at(counts),
                 None if starts is None else at(starts), m, 16, None, None, state, lr, b1, b2, eps, 0.0, step, None,
                 None)

    for bad in (dict(dtype=3), dict(bits=16), dict(tensors=-1), dict(counts=array("q", [-1])), dict(state=511),
                dict(starts=array("q", [256])), dict(starts=array("q", [3])), dict(starts=array("q", [-256])),
                dict(m=None), dict(m=8), dict(bits=8), dict(lr=float("inf")), dict(b1=1.0), dict(b2=-0.1),
                dict(eps=float("nan")), dict(step=0), dict(params=array("q", [0]))):
        with pytest.raises(ValueError):
            step(**bad)
    two, both = array("q", [16, 16]), array("q", [300, 300])
    with pytest.raises(ValueError, match="overlap"):
        step(tensors=2, counts=both, params=two, starts=array("q", [0, 256]), state=4096)
    step(tensors=0)
    size = nat.lib().ictc_gradient_norm_workspace_bytes
    assert size(-1) == -1 and size(1) > 16 and size(121) > size(120)
    for norm, ws, nbytes in ((-1.0, 16, 1 << 20), (float("nan"), 16, 1 << 20), (1.0, None, 1 << 20), (1.0, 16, 64)):
        with pytest.raises(ValueError):
            nat.call("ictc_gradient_norm", 0, 1, at(one), at(n), norm, ws, nbytes, None)


def test_hyperparameters_of_a_group():
    from ictc_o3 import AdamW
    ps = [torch.nn.Parameter(torch.ones(4)) for _ in range(2)]
    for bad in (dict(state_bits=16), dict(betas=(0.9, 1.0)), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            AdamW([dict(params=ps[:1]), dict(params=ps[1:], **bad)])
        opt = AdamW(ps[:1])
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=ps[1:], **bad))
        assert len(opt.param_groups) == 1
