"""Optimizers of the `ocl` device with more than torch's fused ones offer.

``torch.optim.AdamW(params, fused=True)`` and ``torch.optim.Adam(..., fused=True)``
run on this device as they are (one launch over all parameters).  ``AdamW`` here
is the same step with moments that do not follow the parameters' type:

* ``state_bits=32``: fp32 moments for fp32, bf16 or fp16 parameters;
* ``state_bits=8``: moments in 8 bits, a quarter of the memory and of the
  traffic.  Blocks of 256 elements share an fp32 scale; the first moment has a
  sign, 4 bits of exponent and 3 of mantissa, the root of the second moment 4
  bits of exponent and 4 of mantissa.  The step uses the moments before they
  are rounded.

    opt = pytorch_vulkan_b200.optim.AdamW(model.parameters(), lr=1e-3, state_bits=8)
    loss.backward()
    opt.step()
"""
from __future__ import annotations

import torch

from . import _C

_BLOCK = 256
# the state of a parameter by `state_bits`: the two moments, and the scales of 8-bit ones
_KEYS = {
    32: ("exp_avg", "exp_avg_sq"),
    8: ("exp_avg_code", "exp_avg_rms_code", "exp_avg_scale", "exp_avg_rms_scale"),
}


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with fp32 or 8-bit moments, one launch for all parameters of a type.

    The step count of each parameter lives on the device, so that a step
    captured in a ``torch.ocl.Graph`` advances it on every replay (the learning
    rate and the other numbers are those of the capture).  A parameter's first
    step makes its state and cannot be captured.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False,
                 state_bits=32):
        if state_bits not in _KEYS:
            raise ValueError(f"state_bits is 32 or 8, got {state_bits!r}")
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"Invalid betas: {betas}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        self.state_bits = state_bits
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize))

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits}

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        params = self.param_groups[-1]["params"]
        try:
            if len({id(p) for p in params}) != len(params):
                raise ValueError("a parameter is listed twice")
            for p in params:
                if p.device.type != "ocl" or p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                    raise ValueError(
                        f"fp32, bf16 or fp16 parameters on the ocl device expected, got {p.dtype} on {p.device}")
        except ValueError:
            self.param_groups.pop()
            raise

    def _init_state(self, p):
        # whole or not at all: memory may run out on the way
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if self.state_bits == 32:
            for key in _KEYS[32]:
                state[key] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            self.state[p] = state
            return
        n = p.numel()
        for key in _KEYS[8]:
            if not key.endswith("code"):
                state[key] = torch.zeros(-(-n // _BLOCK), dtype=torch.float32, device=p.device)
            elif p.is_contiguous():
                state[key] = torch.zeros(n, dtype=torch.uint8, device=p.device)
            else:  # codes follow the parameter's memory order, which their strides keep
                state[key] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format)
        self.state[p] = state

    def step(self, closure=None):
        # (no graph is recorded below: the update is no torch operation)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            args = (group["params"], self.state, self.state_bits, float(group["lr"]), beta1, beta2, group["eps"],
                    group["weight_decay"], group["maximize"])
            missing = _C.impl_adamw_step(*args)
            if missing:
                if any(_C.impl_graph_capturing(p.device.index) for p in missing):
                    # every replay would begin by zeroing the moments and the step count
                    raise RuntimeError("ocl AdamW: a parameter has no state yet; it needs one step before it is captured")
                for p in missing:
                    self._init_state(p)
                if _C.impl_adamw_step(*args):
                    raise RuntimeError("ocl AdamW: the state of a parameter went away during the step")
        return loss

    @torch.no_grad()
    def write_state_values(self, exp_avgs, exp_avg_sqs):
        """Write the moments that the state holds, as numbers, into fp32 tensors.

        One tensor per parameter that has a state, in the order of
        ``param_groups``, laid out like its parameter (a checkpoint for another
        optimizer, a look at the moments).
        """
        params = [p for group in self.param_groups for p in group["params"]]
        if self.state_bits == 8:
            _C.impl_adamw8_values(params, self.state, exp_avgs, exp_avg_sqs)
            return
        held = [self.state[p] for p in params if self.state.get(p)]
        if len(exp_avgs) != len(held) or len(exp_avg_sqs) != len(held):
            raise ValueError(f"{len(held)} parameters have a state, got {len(exp_avgs)} and {len(exp_avg_sqs)} tensors")
        for s, a, b in zip(held, exp_avgs, exp_avg_sqs):
            a.copy_(s["exp_avg"])
            b.copy_(s["exp_avg_sq"])

    def _fits(self, p, state):
        n, blocks = p.numel(), -(-p.numel() // _BLOCK)
        numels = {"step": 1, "exp_avg": n, "exp_avg_sq": n, "exp_avg_code": n, "exp_avg_rms_code": n,
                  "exp_avg_scale": blocks, "exp_avg_rms_scale": blocks}
        return set(state) == {"step", *_KEYS[self.state_bits]} and all(
            isinstance(v, torch.Tensor) and v.numel() == numels[k]
            and v.dtype == (torch.uint8 if k.endswith("code") else torch.float32) for k, v in state.items())

    def load_state_dict(self, state_dict):
        """As torch's, but the state keeps its own types (torch casts floating state to the parameters'), and one that
        does not fit is refused before anything is replaced."""
        loaded = {}

        def take(_, state_dict):  # after the program's own hooks; torch sees the groups and what belongs to no parameter
            old = [i for group in state_dict["param_groups"] for i in group["params"]]
            new = [p for group in self.param_groups for p in group["params"]]
            for i, p in zip(old, new):
                saved = state_dict["state"].get(i)
                if not saved:
                    continue
                if not self._fits(p, saved):
                    raise ValueError(f"the state of parameter {i} is not one of {self.state_bits} bits that fits it")
                loaded[p] = {k: v.detach().to(device=p.device, copy=True) for k, v in saved.items()}
            ids = set(old)
            return {**state_dict, "state": {k: v for k, v in state_dict["state"].items() if k not in ids}}

        def put(_):  # before the program's own
            self.state.update(loaded)

        hooks = (self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(put, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
