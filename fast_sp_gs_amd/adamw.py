"""AdamW (Adam with decoupled weight decay) over lists of tensors at once, with 32-bit or 8-bit moments, and gradients clipped by the
norm of all of them together. No counterpart in the reference, whose optimisers are `torch.optim.Adam` and its masked form; needed where
networks are regularised by decay, and where learned neighbour logits `sp_W[N, M]` (LBS_method 'W') make the optimiser's moments the
largest thing in memory: 8 bytes an element in 32 bits, 2 in 8.

    m = b1 m + (1 - b1) c g,  v = b2 v + (1 - b2) (c g)^2,  c = min(1, max_norm / (|g| + 1e-6)), NaN if |g| is
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

`adamw_step` and `adamw8_step` step lists of tensors, `AdamW` is the optimiser class over them. Parameters and gradients are float32,
float16 or bfloat16 tensors on one GPU, of any layout without gaps, fewer than 2^34 elements in a call. Tensors that a call writes may not share
memory with any other of its tensors.

8-bit moments: the state of a tensor is one uint8 tensor, blocks of 256 consecutive elements under a power of two each; m with sign, 4
bits of exponent and 3 of fraction, v with 5 and 3. Codes are rounded up or down by a hash of (element, step count, seed) such that
the mean is the value, since changes of a tenth and a thousandth would never reach the next code otherwise. The moments are formed in
float64 from the codes; a code's border counts as reached from 2^-44 of the binade (6e-14) below it on, since decimal betas miss borders that 16-bit
gradients put a moment on. Equal calls give equal results; tensors of a call that have taken as many steps share their random numbers, element by
element. An infinity or a NaN in a moment makes
those of its block of 256 NaN.
"""
from __future__ import annotations

from itertools import chain
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from fast_sp_gs_amd.lib import host

__all__ = ['AdamW', 'adamw_step', 'adamw8_step', 'adamw8_state', 'adamw8_moments', 'adamw8_pack', 'grad_norm']

Rate = Union[float, Sequence[float]]


def _each(value: Rate, n: int) -> List[float]:
    """A number for all tensors, or one for each of them."""
    return [float(v) for v in value] if isinstance(value, (list, tuple)) else [float(value)] * n


def grad_norm(grads: Sequence[Tensor], max_norm: float = float('inf')) -> Tensor:
    """float32 [2] on the device: the 2-norm of all the tensors together, and min(1, max_norm / (norm + 1e-6))."""
    return host.grad_norm(list(grads), float(max_norm))


def _norm(grads, max_norm):
    return None if max_norm is None or not grads else host.grad_norm(grads, float(max_norm))


@torch.no_grad()
def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor],
               steps: Sequence[Tensor], lr: Rate = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: Rate = 1e-8,
               weight_decay: Rate = 1e-2, max_norm: Optional[float] = None) -> Optional[Tensor]:
    """One AdamW step of every tensor, in place; float32 moments in the parameters' layouts. `steps`: how many steps each tensor has
    taken (one-element tensors, all on the host or all float32 on the device; the call adds one). lr, eps and weight_decay: one number, or one
    per tensor. Returns the norm of all gradients together (0-dimensional, on the device) if `max_norm` is given."""
    params, grads = list(params), list(grads)
    n, norm = len(params), _norm(grads, max_norm)
    host.adamw_step(params, grads, list(exp_avgs), list(exp_avg_sqs), list(steps), _each(lr, n), *betas, _each(eps, n),
                    _each(weight_decay, n), norm)
    return None if norm is None else norm[0]


@torch.no_grad()
def adamw8_step(params: Sequence[Tensor], grads: Sequence[Tensor], states: Sequence[Tensor], steps: Sequence[Tensor], lr: Rate = 1e-3,
                betas: Tuple[float, float] = (0.9, 0.999), eps: Rate = 1e-8, weight_decay: Rate = 1e-2,
                max_norm: Optional[float] = None, seed: int = 0) -> Optional[Tensor]:
    """`adamw_step` with both moments of a tensor in one uint8 state (`adamw8_state` makes the first one). `seed` chooses the
    rounding's random numbers together with the step counts."""
    params, grads = list(params), list(grads)
    n, norm = len(params), _norm(grads, max_norm)
    host.adamw8_step(params, grads, list(states), list(steps), _each(lr, n), *betas, _each(eps, n), _each(weight_decay, n), int(seed),
                     norm)
    return None if norm is None else norm[0]


def adamw8_state(param: Tensor) -> Tensor:
    """The 8-bit moments of a tensor that has taken no step."""
    return torch.zeros(host.adamw8_state_bytes(param.numel()), dtype=torch.uint8, device=param.device)


def adamw8_moments(states: Sequence[Tensor], like: Sequence[Tensor], dtype: torch.dtype = torch.float32) -> List[Tuple[Tensor, Tensor]]:
    """(m, v) that the states stand for, in the shapes of the tensors `like` that they belong to. The values have at most four
    significant bits: they are exact in any of the types unless a block's scale takes them out of float16's range. They are parts of one
    allocation."""
    return host.adamw8_moments(list(states), list(like), str(dtype).replace('torch.', ''))


def adamw8_pack(exp_avgs: Sequence[Tensor], exp_avg_sqs: Sequence[Tensor]) -> List[Tensor]:
    """States of float32 moments, rounded to the nearest code."""
    return host.adamw8_pack(list(exp_avgs), list(exp_avg_sqs))


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step on the kernels above. `state_bits` 32: states as torch's AdamW keeps them (checkpoints load either way),
    float32 for parameters of any type; 8: `moments8`, the uint8 state (32-bit checkpoints are taken over, and the other way round).
    `max_norm` clips the gradients by the norm of all of them together within the step, without writing them; `last_norm` then holds that norm.
    `capturable` keeps the step counts on the device, for steps captured into a graph (after a first one that is not); rates are captured as
    they are. The step tells autograd that
    the parameters changed, so `DeformNetwork` packs its weights anew by itself."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, max_norm: Optional[float] = None, capturable: bool = False,
                 seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits must be 8 or 32, got {state_bits}')
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError('lr, eps and weight_decay must not be negative, betas in [0, 1)')
        if max_norm is not None and not max_norm >= 0:
            raise ValueError('max_norm must not be negative')
        self.state_bits, self.max_norm, self.seed, self.last_norm = state_bits, max_norm, seed, None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable))

    def __getstate__(self):  # torch keeps the groups and the states alone
        return dict(super().__getstate__(), state_bits=self.state_bits, max_norm=self.max_norm, seed=self.seed, last_norm=None)

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:  # checkpoints from before torch's AdamW had it
            group.setdefault('capturable', False)

    def _state_of(self, p: Tensor, capturable: bool):
        state = self.state[p]
        if not state:
            if torch.cuda.is_current_stream_capturing():  # every replay would start from zero again
                raise RuntimeError('AdamW: take one step before a step is captured')
            state['step'] = torch.zeros((), dtype=torch.float32, device=p.device if capturable else 'cpu')
            if self.state_bits == 8:
                state['moments8'] = adamw8_state(p)
            else:
                state.update(exp_avg=torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format),
                             exp_avg_sq=torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format))
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # groups of the same betas and counts in the same place go together
        calls, every = {}, []
        for group in self.param_groups:
            params = [p for p in group['params'] if p.grad is not None]
            every += [p.grad for p in params]
            call = calls.setdefault((*group['betas'], group['capturable']), ([], [], [], []))
            call[0].extend(params)
            for rates, key in zip(call[1:], ('lr', 'eps', 'weight_decay')):
                rates.extend([float(group[key])] * len(params))
        if not every:
            return loss
        norm = _norm(every, self.max_norm)
        for (b1, b2, capturable), (params, lr, eps, decay) in calls.items():
            if not params:
                continue
            states = [self._state_of(p, capturable) for p in params]
            grads, steps = [p.grad for p in params], [s['step'] for s in states]
            if self.state_bits == 8:
                host.adamw8_step(params, grads, [s['moments8'] for s in states], steps, lr, b1, b2, eps, decay, self.seed, norm)
            else:
                host.adamw_step(params, grads, [s['exp_avg'] for s in states], [s['exp_avg_sq'] for s in states], steps, lr, b1, b2,
                                eps, decay, norm)
        self.last_norm = None if norm is None else norm[0]
        return loss

    def load_state_dict(self, state_dict):
        """Also a checkpoint with moments of the other width. torch casts what it loads to the parameter's type, which moments do not
        have here: they are taken from the checkpoint itself. 8-bit moments follow the memory: a parameter that takes them over lies as the one
        that they were kept of."""
        if any(group.get('amsgrad') or group.get('maximize') for group in state_dict['param_groups']):
            raise ValueError('AdamW: checkpoints of amsgrad or maximize steps cannot be taken over')
        ids = list(chain.from_iterable(group['params'] for group in state_dict['param_groups']))
        for k, p in zip(ids, chain.from_iterable(group['params'] for group in self.param_groups)):
            for key, t in (state_dict['state'].get(k) or {}).items():
                if key in ('exp_avg', 'exp_avg_sq') and t.shape != p.shape or key == 'moments8' and t.numel() != host.adamw8_state_bytes(p.numel()):
                    raise ValueError(f"AdamW: the checkpoint's {key} has shape {tuple(t.shape)}, which a parameter of {tuple(p.shape)} does not have")
        super().load_state_dict(state_dict)
        own = [(p, group['capturable']) for group in self.param_groups for p in group['params']]
        for k, (p, capturable) in zip(ids, own):
            saved = state_dict['state'].get(k)
            if not saved:
                continue
            state = self.state[p]
            # a count of its own for every parameter, in the place that the group asks for
            state['step'] = torch.as_tensor(saved['step'], dtype=torch.float32).clone().to(p.device if capturable else 'cpu')
            for key in ('exp_avg', 'exp_avg_sq', 'moments8'):
                state.pop(key, None)
            if 'moments8' in saved:
                moments8 = saved['moments8'].to(p.device, copy=True)
                if self.state_bits == 8:
                    state['moments8'] = moments8
                else:
                    (m, v), = adamw8_moments([moments8], [p])
                    state.update(exp_avg=m, exp_avg_sq=v)
            else:
                m, v = (torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(saved[key])
                        for key in ('exp_avg', 'exp_avg_sq'))
                if self.state_bits == 8:
                    state['moments8'], = adamw8_pack([m], [v])
                else:
                    state.update(exp_avg=m, exp_avg_sq=v)
