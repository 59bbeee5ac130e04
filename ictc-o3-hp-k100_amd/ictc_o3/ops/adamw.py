"""AdamW over many tensors at once on HIP kernels, with moments in FP32 or in 8 bits.

A training step of the potential ends in an update of some forty parameters, most of
them small: one launch covers up to 120 tensors.  The moments of all tensors are flat
buffers (``adamw_segments`` says where each tensor's begin); with 8 bits they take two
bytes an element instead of eight.
"""
from __future__ import annotations

from array import array

import torch

from ictc_o3 import _native as nat
from ictc_o3.ops.layer_norm import DTYPES

BLOCK = 256


def adamw_segments(counts):
    """(first element of each tensor's moments, elements of the flat moments) for tensors of these element counts:
    every segment begins at the next multiple of 256."""
    starts, total = [], 0
    for n in counts:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    return starts, total


def _check_moment(t, name, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"adamw: {name} must be a contiguous {dtype} tensor on {device}")


def _check_moments(m, v, ms, vs):
    """Whether the moments are in 8 bits; raises where the four do not belong together."""
    eight, device, held = ms is not None or vs is not None, m.device, m.numel()
    if device.type != "cuda":
        raise ValueError("adamw: tensors must be on a ROCm (cuda) device")
    _check_moment(m, "exp_avg", torch.float8_e4m3fn if eight else torch.float32, device)
    _check_moment(v, "exp_avg_sq", torch.uint8 if eight else torch.float32, device)
    if v.numel() != held:
        raise ValueError("adamw: exp_avg and exp_avg_sq must have as many elements")
    if eight:
        _check_moment(ms, "exp_avg_scale", torch.float32, device)
        _check_moment(vs, "exp_avg_sq_scale", torch.float32, device)
        if held % BLOCK or ms.numel() * BLOCK < held or vs.numel() * BLOCK < held:
            raise ValueError("adamw: 8-bit moments come in blocks of 256 elements with one scale each")
    return eight


class _Lists:
    """Addresses and element counts of parameters and gradients, as the kernels' host arrays."""

    def __init__(self, params, grads, device):
        if len(grads) != len(params):
            raise ValueError("adamw: as many gradients as parameters are needed")
        self.count, dtype, index = len(params), params[0].dtype, device.index
        if dtype not in DTYPES:
            raise ValueError("adamw: parameters must be float32, bfloat16 or float16")
        for p, g in zip(params, grads):
            if (p.dtype is not dtype or g.dtype is not dtype or p.get_device() != index or g.get_device() != index
                    or not p.is_contiguous() or not g.is_contiguous()):
                raise ValueError("adamw: parameters and gradients must be contiguous, of one type and on one device")
        counts = [p.numel() for p in params]
        if [g.numel() for g in grads] != counts:
            raise ValueError("adamw: a gradient must have its parameter's shape")
        self.dtype = DTYPES[dtype]
        self.params = array("q", [p.data_ptr() for p in params])
        self.grads = array("q", [g.data_ptr() for g in grads])
        self.counts = array("q", counts)


def _at(values):
    return None if values is None else values.buffer_info()[0]


def _norm(lists, max_norm, device):
    """ictc_gradient_norm's workspace: [0] the norm, [1] the factor that holds it to max_norm."""
    nbytes = nat.lib().ictc_gradient_norm_workspace_bytes(lists.count)
    ws = torch.empty(nbytes // 4, dtype=torch.float32, device=device)
    nat.call("ictc_gradient_norm", lists.dtype, lists.count, _at(lists.grads), _at(lists.counts), max_norm,
             ws.data_ptr(), nbytes, nat.stream_of(ws))
    return ws


def _step(params, lists, m, v, ms, vs, starts, lr, betas, eps, weight_decay, step, ws):
    nat.call("ictc_adamw_step", lists.dtype, 32 if ms is None else 8, lists.count, _at(lists.params), _at(lists.grads),
             _at(lists.counts), _at(starts), m.data_ptr(), v.data_ptr(), nat.ptr(ms), nat.ptr(vs), m.numel(), lr,
             betas[0], betas[1], eps, weight_decay, step, nat.ptr(ws), nat.stream_of(m))
    # what was read of these tensors before (a graph's saved inputs, transposed copies of a weight) is out of date
    torch.autograd.graph.increment_version([*params, m, v] if ms is None else [*params, m, v, ms, vs])


def adamw_step(params, grads, exp_avg, exp_avg_sq, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               max_norm=None, exp_avg_scale=None, exp_avg_sq_scale=None):
    """One AdamW step of `params` (updated in place) with `grads`, two lists of packed tensors of one type (float32,
    bfloat16 or float16) on one device; `step` counts from 1.

    exp_avg and exp_avg_sq hold the moments of all tensors, flat, laid out by ``adamw_segments``: float32; or, with
    exp_avg_scale and exp_avg_sq_scale (float32, one per 256 elements), float8_e4m3fn and uint8 codes (see
    ``adamw_moments``).  They are updated in place.  Arithmetic is FP32; a parameter of fewer bits is rounded to
    nearest.  With max_norm the gradients are taken as if clipped to that global norm (they are not changed), and the
    norm before clipping is returned as a float32 scalar on the device; otherwise None.  Non-finite gradients make the
    parameters that they reach non-finite."""
    _check_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)
    if max_norm is not None and not max_norm >= 0.0:
        raise ValueError("adamw: max_norm must be zero or more")
    device = exp_avg.device
    if len(params) == 0:
        return None if max_norm is None else torch.zeros((), dtype=torch.float32, device=device)
    lists = _Lists(params, grads, device)
    ws = None if max_norm is None else _norm(lists, max_norm, device)
    _step(params, lists, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, None, lr, betas, eps, weight_decay, step, ws)
    return None if ws is None else ws[0]


def adamw_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, *, dtype=torch.float32):
    """The values of 8-bit moments, (exp_avg, exp_avg_sq) as flat tensors of `dtype`.  They have four significant bits
    at most, so float32 and bfloat16 hold them exactly."""
    if dtype not in DTYPES:
        raise ValueError("adamw: dtype must be float32, bfloat16 or float16")
    if exp_avg_scale is None or exp_avg_sq_scale is None:
        raise ValueError("adamw: moments in 8 bits have scales")
    _check_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)
    n = exp_avg.numel()
    m, v = (torch.empty(n, dtype=dtype, device=exp_avg.device) for _ in range(2))
    nat.call("ictc_adamw_moments", DTYPES[dtype], nat.ptr(exp_avg), nat.ptr(exp_avg_sq), nat.ptr(exp_avg_scale),
             nat.ptr(exp_avg_sq_scale), n, nat.ptr(m), nat.ptr(v), nat.stream_of(exp_avg))
    return m, v


class AdamW(torch.optim.Optimizer):
    """AdamW with torch.optim's interface on ``adamw_step``'s kernels: all parameters of a group in one launch per 120.

    state_bits 32 or 8 chooses the type of the moments.  max_norm bounds the 2-norm over the gradients of all groups;
    the norm before the bound is left in ``grad_norm`` (a device scalar).  A parameter without a gradient is skipped:
    its moments and its count of steps stay as they are."""

    _MOMENTS = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, max_norm=None,
                 state_bits=32):
        if state_bits not in (32, 8):
            raise ValueError("AdamW: state_bits must be 32 or 8")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError("AdamW: betas must be in [0, 1); lr, eps and weight_decay zero or more")
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError("AdamW: max_norm must be zero or more")
        self.max_norm, self.grad_norm, self._flat = max_norm, None, {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits))

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.grad_norm, self._flat = None, {}   # (a copy gathers its moments anew from its per-parameter state)

    def _moments(self, index):
        """The flat moments of a group, whose segments are its parameters' state; made at the first step."""
        if index not in self._flat:
            group = self.param_groups[index]
            ps, eight = group["params"], group["state_bits"] == 8
            starts, total = adamw_segments([p.numel() for p in ps])
            device = ps[0].device
            if eight:
                flat = [torch.zeros(total, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                        torch.zeros(total, dtype=torch.uint8, device=device),
                        torch.ones(total // BLOCK, device=device), torch.ones(total // BLOCK, device=device)]
            else:
                flat = [torch.zeros(total, device=device), torch.zeros(total, device=device), None, None]
            for p, at in zip(ps, starts):
                n, state = -(-p.numel() // BLOCK) * BLOCK, self.state[p]
                state.setdefault("step", 0)
                for name, buffer in zip(self._MOMENTS, flat):
                    if buffer is None:
                        continue
                    per = BLOCK if name.endswith("scale") else 1
                    segment = buffer[at // per:(at + n) // per]
                    if name in state:
                        if state[name].dtype != segment.dtype or state[name].shape != segment.shape:
                            raise ValueError(f"AdamW: the state's {name} does not fit state_bits or its parameter")
                        raw = segment.view(torch.uint8) if segment.element_size() == 1 else segment
                        raw.copy_(state[name].view(raw.dtype))
                    state[name] = segment
            self._flat[index] = (flat, starts)
        return self._flat[index]

    def load_state_dict(self, state_dict):
        """torch.optim's, but the moments keep their type whatever the parameters' is."""
        state = state_dict["state"]
        super().load_state_dict({**state_dict, "state": {}})
        self._flat = {}
        for saved, group in zip(state_dict["param_groups"], self.param_groups):
            for key, p in zip(saved["params"], group["params"]):
                if key in state:
                    self.state[p] = {k: t.to(p.device).clone() if isinstance(t, torch.Tensor) else t
                                     for k, t in state[key].items()}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []   # (group, flat moments, lists, segments, step)
        for index, group in enumerate(self.param_groups):
            flat, starts = self._moments(index) if group["params"] else (None, ())
            by_step = {}
            for p, at in zip(group["params"], starts):
                if p.grad is not None:
                    by_step.setdefault(self.state[p]["step"] + 1, []).append((p, p.grad, at))
            for step, rows in by_step.items():
                if any(g.is_sparse for _, g, _ in rows):
                    raise ValueError("AdamW: gradients must be dense")
                grads = [g.contiguous() for _, g, _ in rows]
                ps = [p for p, _, _ in rows]
                lists = _Lists(ps, grads, flat[0].device)
                work.append((group, flat, lists, array("q", [at for _, _, at in rows]), step, grads, ps))
        ws = None
        if self.max_norm is not None and work:
            if len({w[2].dtype for w in work}) > 1 or len({w[1][0].device for w in work}) > 1:
                raise ValueError("AdamW: max_norm needs parameters of one type on one device")
            every = work[0][2]
            if len(work) > 1:
                every = _Lists([g for w in work for g in w[5]], [g for w in work for g in w[5]], work[0][1][0].device)
            ws = _norm(every, self.max_norm, work[0][1][0].device)
            self.grad_norm = ws[0]
        for group, flat, lists, starts, step, _, ps in work:
            _check_moments(*flat)
            _step(ps, lists, *flat, starts, group["lr"], group["betas"], group["eps"], group["weight_decay"], step, ws)
            for p in ps:
                self.state[p]["step"] = step
        return loss
