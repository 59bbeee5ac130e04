"""AdamW over many tensors at once on HIP kernels, with moments in FP32 or in 8 bits.

A training step of the potential ends in an update of some forty parameters, most of
them small: one launch covers up to 120 tensors.  The moments of all tensors are flat
buffers (``adamw_segments`` says where each tensor's begin); with 8 bits they take two
bytes an element instead of eight.  Checks and launches are in csrc/torch_ops.cpp.
"""
from __future__ import annotations

import operator

import torch

from ictc_o3 import _native as nat

BLOCK = 256


def adamw_segments(counts):
    """(first element of each tensor's moments, elements of the flat moments) for tensors of these element counts:
    every segment begins at the next multiple of 256."""
    starts, total = [], 0
    for n in counts:
        starts.append(total)
        total += -(-n // BLOCK) * BLOCK
    return starts, total


def adamw_step(params, grads, exp_avg, exp_avg_sq, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               max_norm=None, exp_avg_scale=None, exp_avg_sq_scale=None):
    """One AdamW step of `params` (updated in place) with `grads`, two lists of packed tensors of one type (float32,
    bfloat16 or float16) on one device; `step` counts from 1.

    exp_avg and exp_avg_sq hold the moments of all tensors, flat, laid out by ``adamw_segments``: float32; or, with
    exp_avg_scale and exp_avg_sq_scale (float32, one per 256 elements), float8_e4m3fn and uint8 codes (see
    ``adamw_moments``).  They are updated in place.  Arithmetic is FP32; a parameter of fewer bits is rounded to
    nearest.  With max_norm the gradients are taken as if clipped to that global norm (they are not changed), and the
    norm before clipping is returned as a float32 scalar on the device; otherwise None.  Non-finite gradients make the
    parameters that they reach non-finite.  Captured into a graph, the call replays with the `step` and `lr` it had."""
    return nat.ops().adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, step, lr,
                                betas[0], betas[1], eps, weight_decay, max_norm)


def adamw_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, *, dtype=torch.float32):
    """The values of 8-bit moments, (exp_avg, exp_avg_sq) as flat tensors of `dtype`.  They have four significant bits
    at most, so float32 and bfloat16 hold them exactly."""
    if exp_avg_scale is None or exp_avg_sq_scale is None:
        raise ValueError("adamw: moments in 8 bits have scales")
    return nat.ops().adamw_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, dtype)


class AdamW(torch.optim.Optimizer):
    """AdamW with torch.optim's interface on ``adamw_step``'s kernels: all parameters of a group that have one type
    (float32, bfloat16 or float16) in one launch per 120.

    state_bits 32 or 8 chooses the type of the moments.  max_norm bounds the 2-norm over the gradients of all groups;
    the norm before the bound is left in ``grad_norm`` (a device scalar).  A parameter without a gradient is skipped:
    its moments and its count of steps stay as they are.  A group's list of parameters may change between steps,
    and ``state`` may be cleared; its tensors are parts of larger ones, to be changed in place.
    Parameters must be contiguous; a step that is refused changes nothing.  A step cannot be captured into a graph: a
    replay would repeat its count of steps and its learning rate."""

    _MOMENTS = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, max_norm=None,
                 state_bits=32):
        if max_norm is not None and not max_norm >= 0.0:
            raise ValueError("AdamW: max_norm must be zero or more")
        self.max_norm, self.grad_norm, self._flat = max_norm, None, {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits))

    def add_param_group(self, param_group):
        """torch.optim's, with the group's own numbers held to the same ranges as the defaults."""
        g = {**self.defaults, **param_group}
        if g["state_bits"] not in (32, 8):
            raise ValueError("AdamW: state_bits must be 32 or 8")
        if (not all(0.0 <= b < 1.0 for b in g["betas"])
                or not (g["lr"] >= 0 and g["eps"] >= 0 and g["weight_decay"] >= 0)):
            raise ValueError("AdamW: betas must be in [0, 1); lr, eps and weight_decay zero or more")
        super().add_param_group(param_group)

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.grad_norm, self._flat = None, {}   # (a copy gathers its moments anew from its per-parameter state)

    def _moments(self, index):
        """The flat moments of a group, whose segments are its parameters' state.  Made at the first step, and anew from
        that state whenever the group's parameters (which ones, their order, size and device) or its type of moments
        are no longer those that they were made for, or the state was cleared."""
        group = self.param_groups[index]
        ps, eight = group["params"], group["state_bits"] == 8
        counts = list(map(torch.Tensor.numel, ps))
        made_for = (eight, ps[0].device, counts)
        kept = self._flat.get(index)
        if (kept is None or kept[2] != made_for or not all(map(operator.is_, ps, kept[3]))
                or ps[0] not in self.state):
            self._flat.pop(index, None)   # (a fault below leaves the state as the only source)
            starts, total = adamw_segments(counts)
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
            self._flat[index] = (flat, starts, made_for, list(ps))
        return self._flat[index][:2]

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
        if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a step cannot be captured: its count and rate would stay those of the capture")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, stepped = [], []   # (parameters, gradients, flat moments, segments, step, the group's numbers); their states
        for index, group in enumerate(self.param_groups):
            flat, starts = self._moments(index) if group["params"] else (None, ())
            alike = {}   # one step's parameters of one type each
            for p, at in zip(group["params"], starts):
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise ValueError("AdamW: gradients must be dense")
                    state = self.state[p]
                    alike.setdefault((state["step"] + 1, p.dtype), []).append((p, p.grad.contiguous(), at, state))
            for (step, _), rows in alike.items():
                params, grads, segments, states = map(list, zip(*rows))
                work.append((params, grads, *flat, segments, step, group["lr"], *group["betas"], group["eps"],
                             group["weight_decay"]))
                stepped.append((step, states))
        if work:
            norm = nat.ops().adamw_groups(work, self.max_norm)   # (checks all of it before the first launch)
            if norm is not None:
                self.grad_norm = norm
        for step, states in stepped:
            for state in states:
                state["step"] = step
        return loss
