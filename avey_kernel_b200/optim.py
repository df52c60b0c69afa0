"""AdamW over many tensors in one launch (``avey_adamw_v1``).

The reference leaves training to torch; a user who trains through this
package's backward updates the weights here:

* ``adamw_step``: one step over lists of parameters, gradients and states;
* ``AdamW``: a ``torch.optim.Optimizer`` that keeps the states.

For every element, in fp32::

    m = beta1 m + (1 - beta1) g            v = beta2 v + (1 - beta2) g^2
    p = p (1 - lr weight_decay)
          - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)

States are fp32, or 8 bits an element: m and sqrt(v) as ``float8_e4m3fn``
codes in blocks of 256 consecutive elements (in memory order) with one fp32
scale a block (the block's maximum / 448), rounded stochastically from
``(seed, step, element)`` by the rule in ``include/avey_b200.h``: rounding to the
nearest code would never move a second moment that changes by a thousandth a
step, while the codes are 6 to 12 percent apart.

CUDA parameters (fp32, bf16, f16) run natively; CPU parameters take plain
PyTorch, like the rest of the package.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _binding, _native

BLOCK = 256  # elements that share a scale of the 8-bit states
_MASK = 0xffffffff


def state_scales(numel: int) -> int:
    """Scales that the 8-bit states of a tensor of ``numel`` elements need."""
    return -(-numel // BLOCK)


def _memory_order(t: torch.Tensor) -> torch.Tensor:
    """The elements of a dense tensor as a 1-D view in memory order."""
    return t.as_strided((t.numel(),), (1,))


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values of 8-bit states: ``codes`` (of the shape of the
    parameter) times the scale of each block of 256 in memory order."""
    out = torch.empty_like(codes, dtype=torch.float32)
    flat = _memory_order(codes).float()
    _memory_order(out).copy_(flat * scales.repeat_interleave(BLOCK)[:codes.numel()])
    return out


def _quantize(x: torch.Tensor, noise: torch.Tensor):
    """(codes, scales) of the 1-D fp32 values x, from 20-bit noise per element."""
    n = x.numel()
    pad = state_scales(n) * BLOCK - n
    x = torch.nn.functional.pad(x, (0, pad)).view(-1, BLOCK)
    noise = torch.nn.functional.pad(noise, (0, pad)).view(-1, BLOCK).to(torch.int32)
    scale = (x.abs().amax(1, keepdim=True) * (1 / 448)).clamp(min=2.0 ** -126)
    r = x.abs() * (1 / scale)
    small = r < 2.0 ** -6
    bits = torch.where(small, r + 2.0 ** -6, r).view(torch.int32)
    code = ((bits + noise) >> 20) - 960 - 8 * small.to(torch.int32)
    code = code.clamp(max=126) + 128 * (x < 0)
    return code.view(-1)[:n].to(torch.uint8).view(torch.float8_e4m3fn), scale.view(-1)


def _hash(start: int, n: int, seed: int, step: int, device) -> torch.Tensor:
    """The 32-bit hashes of elements start .. start + n - 1 of a call (constants from
    C. Wellons, "Prospecting for hash functions", 2018)."""
    i = torch.arange(start, start + n, device=device)
    key = (seed + 0x9e3779b9 * (step + (i >> 32))) & _MASK
    for mul in (0x7feb352d, 0x846ca68b):
        key = ((key ^ (key >> 16)) * mul) & _MASK
    x = (i & _MASK) ^ key
    x = ((x ^ (x >> 16)) * 0x7feb352d) & _MASK
    x = ((x ^ (x >> 15)) * 0x846ca68b) & _MASK
    return x ^ (x >> 16)


def _check_cpu(i, p, g, m, v, w, scales):
    # A dense tensor, and no other, gives its strides to empty_like.
    if torch.empty_like(p, device='meta').stride() != p.stride() and p.numel() > 1:
        raise ValueError('a parameter must be dense in memory')
    if g.shape != p.shape or g.dtype != p.dtype:
        raise ValueError('a gradient must have the shape and type of its parameter')
    if any(t.dtype != (torch.float8_e4m3fn if scales else torch.float32) for t in (m, v)):
        raise ValueError('states must be float32 or float8_e4m3fn')
    if w is not None and w.dtype != torch.float32:
        raise ValueError(f'masters[{i}] must be float32')
    for t in (m, v) if w is None else (m, v, w):
        if t.shape != p.shape or (t.stride() != p.stride() and p.numel() > 1):
            raise ValueError('states must have the shape and strides of their parameter')
    blocks = state_scales(p.numel())
    for t in scales:
        if t.dtype != torch.float32 or t.numel() != blocks or not t.is_contiguous():
            raise ValueError(f'scales of parameter {i} must be {blocks} contiguous float32 values')


@torch.no_grad()
def _step_cpu(params, grads, exp_avgs, exp_avg_sqs, step, lr, beta1, beta2, eps, weight_decay,
              masters, avg_scales, sq_scales, seed, grad_scale):
    """The step in plain PyTorch (CPU tensors)."""
    n = len(params)
    lists = (grads, exp_avgs, exp_avg_sqs)
    if any(len(x) != n for x in lists) or any(x is not None and len(x) != n
                                              for x in (masters, avg_scales, sq_scales)):
        raise ValueError('every list must hold one tensor for each parameter')
    quant = n > 0 and exp_avgs[0].dtype == torch.float8_e4m3fn
    for i, p in enumerate(params):
        if any((x[i].dtype == torch.float8_e4m3fn) != quant for x in (exp_avgs, exp_avg_sqs)):
            raise ValueError('the states of a step must have one type')
        if quant != (avg_scales is not None) or quant != (sq_scales is not None):
            raise ValueError('exp_avg_scales and exp_avg_sq_scales go with float8_e4m3fn states, '
                             'and only with them')
        _check_cpu(i, p, grads[i], exp_avgs[i], exp_avg_sqs[i], None if masters is None else masters[i],
                   (avg_scales[i], sq_scales[i]) if quant else ())
    start = 0
    for i, p in enumerate(params):
        m, v = exp_avgs[i], exp_avg_sqs[i]
        w = None if masters is None else masters[i]
        # Everything in the memory order of the parameter.
        g = torch.empty_like(p, dtype=torch.float32)
        g.copy_(grads[i])
        g = _memory_order(g)
        if grad_scale is not None:
            g = g * grad_scale
        target = _memory_order(p if w is None else w)
        fm, fv = _memory_order(m), _memory_order(v)
        if quant:
            m32 = _memory_order(dequantize(m, avg_scales[i]))
            v32 = _memory_order(dequantize(v, sq_scales[i])).square()
        else:
            m32, v32 = fm, fv
        m32 = m32 * beta1 + g * (1 - beta1)
        v32 = v32 * beta2 + g * g * (1 - beta2)
        root = v32.sqrt()
        upd = m32 / (root * (1 / math.sqrt(1 - beta2 ** step)) + eps)
        new = target.float() * (1 - lr * weight_decay) - upd * (lr / (1 - beta1 ** step))
        if quant:
            h = _hash(start, p.numel(), seed, step, p.device)
            for x, codes, scales, noise in (
                    (m32, fm, avg_scales[i], ((h & 0xffff) << 4) + 8),
                    (root, fv, sq_scales[i], ((h >> 16) << 4) + 8)):
                if p.numel():
                    c, s = _quantize(x, noise)
                    codes.copy_(c)
                    scales.copy_(s)
        else:
            fm.copy_(m32)
            fv.copy_(v32)
        target.copy_(new)
        if w is not None:
            _memory_order(p).copy_(new)
        start += state_scales(p.numel()) * BLOCK


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
               exp_avgs: Sequence[torch.Tensor], exp_avg_sqs: Sequence[torch.Tensor], *,
               step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, masters: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None, seed: int = 0,
               grad_scale: Optional[torch.Tensor] = None) -> None:
    """One AdamW step, in place, on ``params`` and their states.

    params and grads: fp32, bf16 or f16 (one type a call; on CPU any floating
    type), each parameter dense in memory. exp_avgs, exp_avg_sqs: fp32 moments
    m and v, or ``float8_e4m3fn`` codes of m and sqrt(v) with their fp32 scales
    (``state_scales(numel)`` of them) in exp_avg_scales and exp_avg_sq_scales.
    masters: fp32 copies that carry the update of 16-bit parameters. step: 1
    for the first. grad_scale: one fp32 value on the device that multiplies
    every gradient (a clip factor, the inverse of a loss scale). step, lr and
    seed are host numbers: a captured CUDA graph repeats those of its capture.
    CUDA tensors with forward-mode tangents and calls under a trace raise."""
    if type(step) is not int or step < 1:
        raise ValueError('step must be a whole number, 1 or more')
    beta1, beta2 = betas
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError('betas must be in [0, 1)')
    for name, x in (('lr', lr), ('eps', eps), ('weight_decay', weight_decay)):
        if not math.isfinite(x) or x < 0:
            raise ValueError(f'{name} must be finite and not negative')
    if len(params) and not params[0].is_cuda:
        _step_cpu(params, grads, exp_avgs, exp_avg_sqs, step, lr, beta1, beta2, eps, weight_decay,
                  masters, exp_avg_scales, exp_avg_sq_scales, int(seed) & _MASK, grad_scale)
        return
    status = _binding.module().adamw_step(
        params, grads, exp_avgs, exp_avg_sqs, masters, exp_avg_scales, exp_avg_sq_scales, step, lr,
        beta1, beta2, eps, weight_decay, int(seed) & _MASK, grad_scale)
    if status:
        _native._check(status)


class AdamW(torch.optim.Optimizer):
    """AdamW with its states in 32 or 8 bits, stepping all parameters of a
    group in one launch.

    ``state_bits``: 32 or 8 (see the module). ``master_weights``: keep an fp32
    copy of 16-bit parameters, which carries the update; without it a 16-bit
    parameter is rounded to the nearest value after each step, and updates
    below half a unit in its last place are lost. ``seed`` feeds the 8-bit
    states' rounding."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, *, state_bits: int = 32,
                 master_weights: bool = False, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError('state_bits must be 8 or 32')
        for name, x in (('lr', lr), ('eps', eps), ('weight_decay', weight_decay)):
            if not math.isfinite(x) or x < 0:
                raise ValueError(f'{name} must be finite and not negative')
        if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
            raise ValueError('betas must be two numbers in [0, 1)')
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=bool(master_weights), seed=int(seed)))

    def _init_state(self, p, group):
        state = self.state[p]
        state['step'] = 0
        if group['state_bits'] == 8:
            for name in ('exp_avg', 'exp_avg_sq'):
                state[name] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
                state[name + '_scale'] = torch.zeros(state_scales(p.numel()), device=p.device,
                                                      dtype=torch.float32)
        else:
            for name in ('exp_avg', 'exp_avg_sq'):
                state[name] = torch.zeros_like(p, dtype=torch.float32)
        if group['master_weights'] and p.dtype != torch.float32:
            state['master'] = p.detach().to(torch.float32)

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: Optional[torch.Tensor] = None):
        """One step of every parameter that has a gradient; returns the
        closure's loss, if there is a closure."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        number = 0  # of the call within this step: no two calls round with the same numbers
        for group in self.param_groups:
            # One call per device, type and step count (one in all, ordinarily).
            calls = {}
            for p in group['params']:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError('sparse gradients are not supported')
                state = self.state[p]
                if not state:
                    self._init_state(p, group)
                key = (p.device, p.dtype, state['step'] + 1)
                calls.setdefault(key, []).append((p, state))
            for (_, _, count), members in calls.items():
                def column(name, members=members):
                    return [s[name] for _, s in members] if name in members[0][1] else None
                adamw_step([p for p, _ in members], [p.grad for p, _ in members],
                           column('exp_avg'), column('exp_avg_sq'), step=count, lr=float(group['lr']),
                           betas=group['betas'], eps=group['eps'],
                           weight_decay=group['weight_decay'], masters=column('master'),
                           exp_avg_scales=column('exp_avg_scale'),
                           exp_avg_sq_scales=column('exp_avg_sq_scale'),
                           seed=group['seed'] + 0x632be5ab * number, grad_scale=grad_scale)
                for _, state in members:  # once the step has been taken
                    state['step'] = count
                number += 1
        return loss

    def load_state_dict(self, state_dict):
        """As in torch, but the states keep their own types (torch casts them
        to the parameter's, which would round fp32 states of 16-bit
        parameters and decode 8-bit ones). States of a parameter whose layout in
        memory has changed follow it; 8-bit ones, whose blocks go by that layout,
        are rounded to the nearest codes of their new blocks."""
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict['param_groups'] for i in g['params']]
        params = [p for g in self.param_groups for p in g['params']]
        for i, p in zip(ids, params):
            saved = state_dict['state'].get(i, {})
            state = self.state[p]
            for name, value in saved.items():
                if isinstance(value, torch.Tensor):
                    state[name] = value.detach().to(p.device, copy=True)
            for name in ('exp_avg', 'exp_avg_sq', 'master'):
                old = state.get(name)
                if old is None or old.stride() == p.stride() or old.shape != p.shape:
                    continue
                if old.dtype != torch.float8_e4m3fn:
                    state[name] = torch.empty_like(p, dtype=old.dtype).copy_(old)
                    continue
                value = torch.empty_like(p, dtype=torch.float32)
                value.copy_(dequantize(old, state[name + '_scale']))
                half = torch.full((p.numel(),), 1 << 19, device=p.device)
                codes, state[name + '_scale'] = _quantize(_memory_order(value), half)
                state[name] = torch.empty_like(p, dtype=old.dtype)
                _memory_order(state[name]).copy_(codes)
