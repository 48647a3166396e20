"""Muon: momentum whose matrix updates are orthogonalised (``newton_schulz``),
for the hidden 2-D parameters; embeddings, the output head, biases and norm
gains stay with AdamW (``lm.build_optimizer``). The reference trains with AdamW
only (train.py:851-859)."""

from __future__ import annotations

import torch

from .training_ops import DEFAULT_COEFFICIENTS, newton_schulz


class Muon(torch.optim.Optimizer):
    """For each matrix W [m, n] with gradient g (m = fan-out):
        buf <- momentum buf + g
        u = g + momentum buf (nesterov) or buf
        W <- (1 - lr weight_decay) W - lr 0.2 sqrt(max(m, n)) newton_schulz(u)
    The factor gives the update the size of an AdamW step (rms about 0.2), so
    one learning rate serves both optimisers."""

    def __init__(self, params, lr: float = 3e-4, momentum: float = 0.95, weight_decay: float = 0.1,
                 nesterov: bool = True, steps: int = 5, coefficients=DEFAULT_COEFFICIENTS) -> None:
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0 or steps < 1:
            raise ValueError(f"Muon: bad hyper-parameters lr={lr} momentum={momentum} weight_decay={weight_decay} "
                             f"steps={steps}")
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      coefficients=tuple(coefficients)))

    def add_param_group(self, group: dict) -> None:
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise ValueError(f"Muon updates matrices; got a parameter of shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            grads = [p.grad for p in params]
            for p, g in zip(params, grads):
                if "momentum_buffer" not in self.state[p]:
                    self.state[p]["momentum_buffer"] = torch.zeros_like(g)
            bufs = [self.state[p]["momentum_buffer"] for p in params]
            torch._foreach_mul_(bufs, group["momentum"])
            torch._foreach_add_(bufs, grads)
            us = torch._foreach_add(grads, bufs, alpha=group["momentum"]) if group["nesterov"] else bufs
            updates = newton_schulz(us, steps=group["steps"], coefficients=group["coefficients"])
            if group["weight_decay"]:
                torch._foreach_mul_(params, 1.0 - group["lr"] * group["weight_decay"])
            for p, u in zip(params, updates):
                p.add_(u, alpha=-group["lr"] * 0.2 * max(p.shape) ** 0.5)
        return loss


class OptimizerPair(torch.optim.Optimizer):
    """Optimisers over disjoint parameters that step together, as one optimiser:
    its groups and states are theirs, so that schedulers and gradient scalers
    take it. state_dict is the list of theirs. Groups are added to one of them."""

    def __init__(self, *optimizers: torch.optim.Optimizer) -> None:
        self.optimizers = optimizers
        self._made = False
        super().__init__([g for o in optimizers for g in o.param_groups], {})
        self._made = True

    # the base class's own copies are never set: a loaded optimiser has new ones
    @property
    def param_groups(self) -> list[dict]:
        return [g for o in self.optimizers for g in o.param_groups]

    @param_groups.setter
    def param_groups(self, groups) -> None:
        pass

    @property
    def state(self) -> dict:
        return {p: s for o in self.optimizers for p, s in o.state.items()}

    @state.setter
    def state(self, state) -> None:
        pass

    def add_param_group(self, group: dict) -> None:
        if self._made:
            raise RuntimeError("OptimizerPair: add the group to one of its optimizers")

    def __getstate__(self) -> dict:
        return {"optimizers": self.optimizers}

    def __setstate__(self, state: dict) -> None:
        self.__init__(*state["optimizers"])

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for o in self.optimizers:
            o.step()
        return loss

    def zero_grad(self, set_to_none: bool = True) -> None:
        for o in self.optimizers:
            o.zero_grad(set_to_none=set_to_none)

    def state_dict(self) -> list[dict]:
        return [o.state_dict() for o in self.optimizers]

    def load_state_dict(self, state: list[dict]) -> None:
        if len(state) != len(self.optimizers):
            raise ValueError(f"OptimizerPair: {len(state)} states for {len(self.optimizers)} optimisers")
        for o, s in zip(self.optimizers, state):
            o.load_state_dict(s)
