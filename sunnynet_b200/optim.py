"""AdamW as a torch optimiser over ``kernels.adamw_step``: the optimiser of the
reference's training loop (train/train.py:171-359), updating all of a group's
tensors in one launch, with states in 32 or 8 bits."""
from __future__ import annotations

import collections

import torch

from . import kernels

__all__ = ["AdamW"]


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay. ``state_bits=8`` keeps both moments
    as float8_e4m3fn codes with a scale for each ``kernels.STATE_BLOCK`` values
    (2.03 bytes a parameter instead of 8). Parameters are contiguous tensors on
    a GPU. The step number lives on the host: to capture a step into a CUDA
    graph, call ``kernels.adamw_step`` with a step tensor. ``max_norm``: gradients
    whose common norm (of all groups) is larger are scaled to it as the step reads
    them, .grad stays as it is; ``grad_norm`` is then the last step's norm, on the GPU.
    All gradients are then on one GPU; a state dict does not hold ``max_norm``."""

    max_norm = grad_norm = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
                 state_bits=32, max_norm=None):
        if max_norm is not None and not max_norm >= 0:
            raise ValueError("AdamW: max_norm must not be negative")
        if state_bits not in (8, 32):
            raise ValueError("AdamW: states have 8 or 32 bits")
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0):
            raise ValueError("AdamW: lr, eps and weight_decay must not be negative")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError("AdamW: betas are in [0, 1)")
        self.max_norm = max_norm
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits))

    def __getstate__(self):
        return {**super().__getstate__(), "max_norm": self.max_norm}

    def _state(self, p, bits):
        s = self.state[p]
        if not s:
            kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
            s["step"] = 0
            # zero bytes are zero in either type
            for k in ("exp_avg", "exp_avg_sq"):
                s[k] = torch.zeros(p.shape, dtype=torch.float32 if bits == 32 else torch.uint8,
                                   device=p.device).view(kind)
            if bits == 8:
                blocks = -(-p.numel() // kernels.STATE_BLOCK)
                for k in ("avg_scale", "sq_scale"):
                    s[k] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step in a capture would repeat one step number: call "
                               "kernels.adamw_step with a step tensor")
        factor = None
        if self.max_norm is not None:
            grads = [p.grad for group in self.param_groups for p in group["params"] if p.grad is not None]
            if grads:
                grads = [g if g.layout != torch.strided else g.contiguous() for g in grads]
                self.grad_norm, factor = kernels.grad_norm(grads, self.max_norm)
        for group in self.param_groups:
            bits = group["state_bits"]
            alike = collections.defaultdict(list)  # one call takes one kind of tensors
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                s = self._state(p, bits)
                alike[p.device, p.dtype, p.grad.dtype, s["step"] + 1].append((p, s))
            for (_, _, _, t), these in alike.items():
                pick = lambda k: [s[k] for _, s in these]  # noqa: B023,E731
                kernels.adamw_step(
                    [p for p, _ in these], [p.grad.contiguous() for p, _ in these],
                    pick("exp_avg"), pick("exp_avg_sq"), t, group["lr"], *group["betas"],
                    group["eps"], group["weight_decay"],
                    pick("avg_scale") if bits == 8 else None,
                    pick("sq_scale") if bits == 8 else None, factor)
                for _, s in these:
                    s["step"] = t
        return loss

    def load_state_dict(self, state_dict):
        """A state dict of this class or of torch.optim.AdamW (states of 32 bits,
        kept in float32 here). One that asks for what this class does not do
        (maximize, amsgrad, weight decay that is not decoupled, states of 8 bits
        where it has none) is refused, and nothing is changed."""
        for mine, g in zip(self.param_groups, state_dict["param_groups"]):
            if g.get("maximize") or g.get("amsgrad") or \
                    (g.get("weight_decay") and not g.get("decoupled_weight_decay", True)):
                raise ValueError("AdamW: maximize, amsgrad and weight decay that is not decoupled "
                                 "are not supported")
            if "state_bits" not in g and mine["state_bits"] != 32:
                raise ValueError("AdamW: this optimiser has states of 8 bits, the state dict of 32")
        super().load_state_dict(state_dict)
        for g in self.param_groups:
            g.setdefault("state_bits", 32)
        # torch gives states their parameter's type: put back the saved ones
        for g, saved in zip(self.param_groups, state_dict["param_groups"]):
            wide = ("exp_avg", "exp_avg_sq") if g["state_bits"] == 32 else ()  # torch's may be narrower
            for p, i in zip(g["params"], saved["params"]):
                if i in state_dict["state"]:
                    self.state[p] = {k: int(v) if k == "step" else
                                     v.detach().to(p.device, torch.float32 if k in wide else v.dtype,
                                                   copy=True).contiguous()
                                     if isinstance(v, torch.Tensor) else v
                                     for k, v in state_dict["state"][i].items()}
