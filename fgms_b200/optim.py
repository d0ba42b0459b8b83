"""AdamW for the networks of this package: one launch for parameters that take their steps together, moments in 32 or in 8 bits.

The layers leave gradients (``nn``, ``unet.UNetStep``); this is what takes a step with them.  The kernel is
``backend.fgms_adamw_cuda`` (``csrc/adamw.cuh``).
"""
from __future__ import annotations

from collections import Counter

import torch

from . import backend

__all__ = ["AdamW"]

_BLOCK = 128  # values that share a scale


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay, ``w -= lr * (weight_decay * w + m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps))``.

    ``state_bits=8`` keeps both moments as e4m3 codes with a float32 scale for each 128 values, a quarter of the memory and of the
    traffic; codes are rounded at random, reproducibly for a ``seed``.  float16 and bfloat16 parameters get a float32 ``master`` copy, without
    which updates of less than half a step of their type are lost, unless ``master=False``; whoever else writes such a parameter writes
    ``state[p]["master"]`` too, as the next step starts from that.  Works in a captured graph (the steps are
    counted on the device; ``lr`` may be a float32 tensor of one value there) and with ``torch.amp.GradScaler``, whose scale and verdict
    the kernel reads.  Before a capture every parameter must have taken a step, as its state would be made anew by every replay; after it the graph works on
    the state there is: ``load_state_dict`` makes another, and a step outside the graph has to be taken by the same parameters.  Parameters must
    be contiguous CUDA tensors; a parameter without a gradient is passed over.  No sparse gradients, no ``amsgrad``, no ``maximize``.

    The parameters of a group that have all taken the same steps share the count of them, and a launch for each 400.  Those that miss a step have a
    count and a launch of their own from then on, also if the others miss one later; only ``load_state_dict`` brings equal counts together."""

    _step_supports_amp_scaling = True  # GradScaler hands over its scale and what it found instead of waiting for the device

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits: int = 32, master: bool = True, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 32 or 8, got {state_bits}")
        if not isinstance(lr, torch.Tensor) and not 0.0 <= lr < float("inf"):
            raise ValueError(f"lr must be finite and not negative, got {lr}")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not 1e-37 <= eps < float("inf") or not 0.0 <= weight_decay < float("inf"):
            raise ValueError(f"eps must be at least 1e-37 and weight_decay not negative, got {eps}, {weight_decay}")
        if not 0 <= seed < 2 ** 32:
            raise ValueError("seed must be in [0, 2^32)")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, master=master, seed=seed))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                raise ValueError(f"parameters must be float32, float16 or bfloat16, got {p.dtype}")

    def _init_state(self, group, p, step):
        s = self.state[p]
        s["step"] = step
        if group["state_bits"] == 8:
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                s[name + "_scale"] = torch.zeros((p.numel() + _BLOCK - 1) // _BLOCK, dtype=torch.float32, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["master"] and p.dtype != torch.float32:
            s["master"] = p.detach().to(torch.float32, copy=True, memory_format=torch.contiguous_format)

    @staticmethod
    def _not_in_a_capture():
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured step needs parameters that have all taken the same steps before the capture: their state would be made "
                               "anew by every replay")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grad_scale, found_inf = getattr(self, "grad_scale", None), getattr(self, "found_inf", None)
        # Parameters that have taken the same steps share the tensor that counts them, and a launch.
        sharing = Counter(id(s["step"]) for s in self.state.values() if "step" in s)
        for group in self.param_groups:
            calls, fresh = {}, {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("AdamW takes no sparse gradients")
                if not p.is_cuda or not p.is_contiguous():
                    raise ValueError("parameters must be contiguous CUDA tensors")
                if "step" not in self.state[p]:
                    self._not_in_a_capture()
                    if p.device not in fresh:
                        fresh[p.device] = torch.zeros(2, dtype=torch.int32, device=p.device)
                    self._init_state(group, p, fresh[p.device])
                    sharing[id(fresh[p.device])] += 1
                calls.setdefault(id(self.state[p]["step"]), []).append(p)
            for key, params in calls.items():
                states = [self.state[p] for p in params]
                step = states[0]["step"]
                if sharing[key] != len(params):  # the others do not take this step
                    self._not_in_a_capture()
                    step = step.clone()
                    for s in states:
                        s["step"] = step
                lists = {name: [s[name] for s in states] for name in states[0] if name not in ("step", "master")}
                masters = [s.get("master") for s in states]
                on = lambda t: t if t is None or t.device == step.device else t.to(step.device)
                backend.fgms_adamw_cuda(params, [p.grad.contiguous() for p in params], lists["exp_avg"], lists["exp_avg_sq"], step, group["lr"],
                                        group["betas"][0], group["betas"][1], group["eps"], group["weight_decay"],
                                        masters=masters if any(m is not None for m in masters) else None,
                                        exp_avg_scales=lists.get("exp_avg_scale"), exp_avg_sq_scales=lists.get("exp_avg_sq_scale"),
                                        seed=group["seed"], grad_scale=on(grad_scale), found_inf=on(found_inf))
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """The base class would cast the moments and masters to the parameters' type: they are taken as they were saved."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        counted = {}
        for i, (k, p) in zip(saved, ((k, p) for k, g in enumerate(self.param_groups) for p in g["params"])):
            if i not in state_dict["state"]:
                continue
            s = self.state[p]
            for name, value in state_dict["state"][i].items():
                s[name] = value.to(device=p.device, copy=True) if isinstance(value, torch.Tensor) else value
            # parameters of a group that have taken the same steps share their count again
            key = (k, p.device, int(s["step"][0]))
            s["step"] = counted.setdefault(key, s["step"])
