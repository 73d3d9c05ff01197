"""AdamW over many tensors at once, with states in 32 or in 8 bits, clipped by the norm of all gradients without a wait of
the host. No counterpart in the reference, whose optimizer is `FusedAdam` (one float32 tensor per group, no weight decay).
"""
from __future__ import annotations

import copy
import math
from typing import Any, Callable, Iterable, Sequence

import torch

from . import _native


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay): per element, c the clipping coefficient and t the parameter's step,

        g = c grad, m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr wd) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

    in 32 bits, p rounded once to its type. Parameters and gradients are contiguous float32, bfloat16 or float16 GPU tensors
    (a gradient that is not contiguous is copied); a launch takes 60 to 72 tensors, of up to 8 groups.

    lr, betas, eps, weight_decay, state_bits: defaults that a group may override. `lr` is a float or a list of up to 7 rates
    cycled over the last dimension's columns, as `FusedAdam` has them.

    state_bits 32: states `exp_avg` and `exp_avg_sq` (float32), as torch.optim.AdamW names them. 8: m / sqrt(v) and sqrt(v) as
    bytes `exp_avg_ratio` and `exp_avg_sq_root` with one float per 256 elements (`root_scale`; the codes are described in
    efgs.h), rounded by a dither from (element, step, seed) so that they are right in the mean; 16 bytes of traffic an
    element and step for float32 parameters in place of 28. They need beta1^2 < beta2. `moments` reads either as float32.

    max_grad_norm: if set, gradients count times min(1, max_grad_norm / (norm + 1e-6)), norm over all gradients of the step (they
    themselves stay as they are); where the norm is not finite, parameters and moments stay as they are (8-bit ones to their codes,
    where the betas have changed). The
    norm is read on the device and left in `grad_norm` (a tensor of no dimensions; None before the first such step).

    The step count is the host's, so a step cannot be captured into a graph, and t counts calls: a step left out for its norm too, whose
    norm the host does not wait for. Moments of fewer gradients than t are then corrected as of t: after k steps left out
    from the start, the default betas make the first update 0.74 (k = 1), 0.48 (10) and, past thousands, up to 3.2 times lr, and the
    difference fades as the moments fill. A program that reads `grad_norm` may set the states' `step` back.

    8-bit states belong to their tensor as it is laid out: a scale stands for 256 consecutive elements. Rows that are selected, moved
    or appended (densification, pruning) tear codes from their scales: hold such tensors in groups of state_bits 32, or drop
    their entries of `state` with the change, which begins them anew. `moments` decodes, nothing encodes.
    """

    def __init__(self, params: Iterable, lr: float | Sequence[float] = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_grad_norm: float | None = None, seed: int = 0) -> None:
        _check_max_norm(max_grad_norm)
        self.max_grad_norm = max_grad_norm
        self.seed = int(seed)
        self.grad_norm: torch.Tensor | None = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def __getstate__(self) -> dict[str, Any]:
        # (of an optimizer the base class copies and pickles its groups and states alone)
        return {**super().__getstate__(), 'max_grad_norm': self.max_grad_norm, 'seed': self.seed, 'grad_norm': self.grad_norm}

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        super().add_param_group(param_group)
        try:
            _check_group(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise

    def step(self, closure: Callable[[], Any] | None = None) -> Any:
        """One step of every parameter that has a gradient; returns what `closure` (re-evaluated first, if given) returns."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.grad_norm = _native.adamw_step(self.param_groups, self.state, self.max_grad_norm, self.seed & 0xffffffff)
        return loss

    def moments(self, params: torch.Tensor | Sequence[torch.Tensor]) -> Any:
        """(exp_avg, exp_avg_sq) in float32 of a parameter, or a list of them for a sequence of parameters: 32-bit states
        themselves, new tensors for 8-bit ones."""
        if isinstance(params, torch.Tensor):
            return _native.adamw_moments([params], self.state)[0]
        return _native.adamw_moments(list(params), self.state)

    def state_dict(self) -> dict[str, Any]:
        """The base class's entries, and `seed` and `max_grad_norm`."""
        return {**super().state_dict(), 'seed': self.seed, 'max_grad_norm': self.max_grad_norm}

    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """Goes on where the saved optimizer stood: with its groups' values, and its `seed` and `max_grad_norm` if they are saved.
        torch.optim.AdamW's saved states are taken too (as 32-bit ones), not with amsgrad or maximize."""
        loaded: dict[str, Any] = {}

        def take(_: AdamW, given: dict[str, Any]) -> dict[str, Any]:
            _check_max_norm(given.get('max_grad_norm'))
            loaded.update(given, param_groups=[{'state_bits': 32, **g} for g in given['param_groups']])
            for group in loaded['param_groups']:
                _check_group(group)
            return loaded

        # behind the hooks that a program has registered, and before those that it has for the end
        hooks = [self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(lambda _: self._take_states(loaded), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_states(self, loaded: dict[str, Any]) -> None:
        # (the base class casts every floating state to its parameter's type, and bytes too)
        self.seed = int(loaded.get('seed', self.seed))
        self.max_grad_norm = loaded.get('max_grad_norm', self.max_grad_norm)
        saved_ids = [i for g in loaded['param_groups'] for i in g['params']]
        params = [p for g in self.param_groups for p in g['params']]
        for i, p in zip(saved_ids, params):
            if i not in loaded['state']:
                continue
            own = {}
            for key, value in loaded['state'][i].items():
                if key == 'step':
                    own[key] = int(value)
                elif isinstance(value, torch.Tensor):
                    own[key] = value.detach().to(p.device).clone(memory_format=torch.contiguous_format)
                else:
                    own[key] = copy.deepcopy(value)
            self.state[p] = own


def _check_max_norm(max_grad_norm: float | None) -> None:
    if max_grad_norm is not None and not max_grad_norm > 0.0:
        raise ValueError(f'efgs: max_grad_norm must be positive, got {max_grad_norm}')


def _number(name: str, value: Any) -> float:
    try:
        if not isinstance(value, str):  # (which the step does not take)
            return float(value)
    except (TypeError, ValueError, RuntimeError):
        pass
    raise ValueError(f'efgs: {name} must be a number, got {value!r}')


def _check_group(group: dict[str, Any]) -> None:
    # (a launch's blocks update all tensors at once)
    if len({id(p) for p in group['params']}) != len(group['params']):
        raise ValueError('efgs: a parameter group holds a parameter more than once')
    for key in ('lr', 'betas', 'eps', 'weight_decay', 'state_bits'):
        if key not in group:
            raise ValueError(f'efgs: a parameter group lacks {key}')
    # (of saved groups of torch's optimizers)
    if group.get('amsgrad') or group.get('maximize') or group['weight_decay'] and not group.get('decoupled_weight_decay', True):
        raise ValueError('efgs: AdamW has no amsgrad, no maximize and no weight decay through the gradient')
    lr, betas = group['lr'], group['betas']
    rates = lr if isinstance(lr, (list, tuple)) else [lr]
    if not 1 <= len(rates) <= 7:
        raise ValueError('efgs: between 1 and 7 learning rates are supported')
    if not all(math.isfinite(_number('lr', rate)) for rate in rates):
        raise ValueError(f'efgs: learning rates must be finite, got {lr}')
    if not isinstance(betas, (list, tuple)) or len(betas) != 2:
        raise ValueError(f'efgs: betas must be two numbers, got {betas}')
    beta1, beta2 = (_number('betas', b) for b in betas)
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f'efgs: betas must lie in [0, 1), got {(beta1, beta2)}')
    if not 0.0 <= _number('eps', group['eps']) < math.inf:
        raise ValueError(f'efgs: eps must be finite and not negative, got {group["eps"]}')
    if not math.isfinite(_number('weight_decay', group['weight_decay'])):
        raise ValueError(f'efgs: weight_decay must be finite, got {group["weight_decay"]}')
    if group['state_bits'] not in (8, 32):
        raise ValueError(f'efgs: state_bits must be 32 or 8, got {group["state_bits"]}')
    if group['state_bits'] == 8 and not beta1 * beta1 < beta2:
        raise ValueError(f'efgs: 8-bit states need beta1^2 < beta2, got {(beta1, beta2)}')


def grad_norm(tensors: torch.Tensor | Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm over all elements of `tensors` (float32, bfloat16 or float16 on one GPU device) as a float32 tensor of no
    dimensions: summed in 64 bits in a fixed order, without a wait of the host. Not differentiable: the result is no part of a graph."""
    return _native.grad_norm([tensors] if isinstance(tensors, torch.Tensor) else list(tensors))
