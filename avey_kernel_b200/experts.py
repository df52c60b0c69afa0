"""A mixture of experts: routing, the rows' way to their experts and back, and the
experts' linear layers with ragged row counts.

``expert_linear(x, weight, offsets, bias)`` multiplies the rows
``[offsets[e], offsets[e + 1])`` of x by expert e's weights: the position-wise
layers of a mixture of experts (``layers.residual_linear`` is the dense form),
native in both directions (``avey_linear_fwd_v1``, ``avey_linear_bwd_v1``).
Around it::

    weights, chosen = route(logits, k)            # each token's k experts
    slots, offsets = arrange(chosen, experts)     # their places, sorted by expert
    h = expert_linear(dispatch(x, slots), w, offsets, b, activation='relu2')
    y = combine(expert_linear(h, ...), slots, weights, residual=x)

``group_by_expert`` sorts tokens that have one expert each. Row counts stay on
the device: no call waits for the GPU, so all can be captured in a CUDA graph.

The reference has no counterpart ("Avey-B's static layers are ordinary matrix
multiplications and are outside this module", avey_kernels/ops.py:1-7).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import _binding, _native
from .layers import _ACT_IDS, _act_torch, _check_act

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def group_by_expert(experts: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(order, offsets)`` for a 1-D tensor of expert numbers in
    [0, num_experts): ``order`` sorts the entries by expert (entries of one
    expert in their given order), ``offsets`` (int32, num_experts + 1) bounds
    each expert's run in it."""
    if experts.ndim != 1 or experts.dtype not in (torch.int32, torch.int64):
        raise ValueError('experts must be a 1-D tensor of int32 or int64 expert numbers')
    order = torch.argsort(experts, stable=True)
    bounds = torch.arange(num_experts + 1, device=experts.device, dtype=experts.dtype)
    offsets = torch.searchsorted(experts[order], bounds, out_int32=True)
    return order, offsets


def _expert_linear_torch(x, weight, offsets, bias, activation):
    """The plain PyTorch form (CPU tensors), with the native form's reading of
    the offsets: out of order or out of range they are pulled into range."""
    rows, parts, end = x.shape[0], [], 0
    for e, bound in enumerate(offsets[1:].tolist()):
        start, end = end, min(max(bound, end), rows)
        y = F.linear(x[start:end], weight[e], None if bias is None else bias[e])
        parts.append(_act_torch(y, activation))
    parts.append(x.new_zeros(rows - end, weight.shape[1]))
    return torch.cat(parts)


def expert_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                  bias: Optional[torch.Tensor] = None, *, activation: str = 'identity'
                  ) -> torch.Tensor:
    """``act(x W_e^T + b_e)`` for every row of expert e's group.

    x ``[rows, d_in]`` with the rows of an expert next to each other, weight
    ``[experts, d_out, d_in]``, offsets int32 ``[experts + 1]`` on x's device
    (``offsets[0] = 0``, rising; an expert may have no row), bias ``[experts,
    d_out]``. Rows from ``offsets[-1]`` on belong to no expert: they give
    zeros and get zero gradients. The gradients of experts without rows are
    zero. bf16 / f16 CUDA tensors of one dtype run natively (forward-mode tangents
    and traces raise); CPU tensors take plain PyTorch."""
    _check_act(activation)
    if x.is_cuda:
        return _binding.module().linear(x, weight, bias, None, offsets, _ACT_IDS[activation],
                                        _native.LINEAR_AUTO)
    if x.ndim != 2 or weight.ndim != 3 or weight.shape[2] != x.shape[1]:
        raise ValueError('x must be [rows, d_in] and weight [experts, d_out, d_in]')
    if bias is not None and bias.shape != weight.shape[:2]:
        raise ValueError('bias must have shape [experts, d_out]')
    if offsets.shape != (weight.shape[0] + 1,) or offsets.dtype != torch.int32:
        raise ValueError(f'offsets must be {weight.shape[0] + 1} contiguous int32 values')
    return _expert_linear_torch(x, weight, offsets, bias, activation)


# ------------------------------------------------------------------ routing

def route(logits: torch.Tensor, k: int, *, bias: Optional[torch.Tensor] = None,
          score: str = 'softmax', groups: int = 1, top_groups: int = 1, group_best: int = 1,
          renormalize: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(weights, chosen)``: the k experts of each token and what their results count.

    logits ``[..., experts]`` (fp32, bf16 or f16; up to 1024 experts, k up to 32).
    Scores s are the softmax of a token's logits or, with ``score='sigmoid'``, their
    logistic function. Experts rank by their logits, or with ``bias`` (fp32
    ``[experts]``, which balances the experts' loads and has no gradient) by ``s +
    bias``. With ``groups`` > 1 (consecutive experts, up to 32 groups) only those of the
    best ``top_groups`` groups are chosen from; a group ranks by the sum of the ranks of
    its best ``group_best`` experts (1 or 2; for 2 without a bias, of their scores).
    Ties go to the lowest index. ``chosen`` (int32 ``[..., k]``) has them from the best on,
    ``weights`` (fp32 ``[..., k]``) are ``scale * s``, divided by the sum of the chosen
    scores with ``renormalize``.

    The choice is the formula's also where scores are nearer than fp32 tells. A logit of
    -inf takes an expert out: it ranks below all others and its weight is 0 (zeros for a
    token whose logits all are). NaN ranks last; it or +inf makes a softmax NaN, in its weights
    and their gradients, and NaN a sigmoid where it is chosen.

    CUDA tensors run natively, forward and backward (the weights' gradient goes to the
    logits); forward-mode tangents, traces and second differentiation raise. CPU
    tensors take plain PyTorch."""
    if score not in _native.SCORE_IDS:
        raise ValueError("score must be 'softmax' or 'sigmoid'")
    if logits.is_cuda:
        return _binding.module().route(logits, bias, k, _native.SCORE_IDS[score], groups, top_groups,
                                       group_best, renormalize, scale)
    if logits.ndim < 1 or logits.dtype not in _FLOATS or not 1 <= logits.shape[-1] <= _native.MAX_EXPERTS:
        raise ValueError('logits must be [..., experts] in float32, float16 or bfloat16, with 1 to '
                         f'{_native.MAX_EXPERTS} experts')
    experts = logits.shape[-1]
    if not 1 <= groups <= _native.MAX_GROUPS or experts % groups or not 1 <= top_groups <= groups:
        raise ValueError(f'groups must divide the experts and be 1 to {_native.MAX_GROUPS}, top_groups 1 to groups')
    if group_best not in (1, 2):
        raise ValueError('group_best must be 1 or 2')
    if not 1 <= k <= min(_native.MAX_CHOICES, experts // groups * top_groups):
        raise ValueError(f'k must be 1 to {_native.MAX_CHOICES} and no more than the experts to choose from')
    if bias is not None and (bias.shape != (experts,) or bias.dtype != torch.float32):
        raise ValueError('bias must be float32 of shape [experts]')
    if not math.isfinite(scale):
        raise ValueError('scale must be finite')
    return _route_torch(logits, k, bias, score, groups, top_groups, group_best, renormalize, scale)


def _route_torch(logits, k, bias, score, groups, top_groups, group_best, renormalize, scale):
    """The plain PyTorch form (CPU tensors)."""
    with torch.no_grad():
        z = logits.double()
        out = z == -math.inf
        exact = torch.sigmoid(z) if score == 'sigmoid' else torch.softmax(z, -1)
        rank = z if bias is None else exact + bias.double()
        by = exact if bias is None and group_best == 2 else rank
        last = rank.isnan()
        rank, by = (torch.where(out, -math.inf, t).nan_to_num(-math.inf, posinf=math.inf, neginf=-math.inf)
                    for t in (rank, by))
        if groups > 1:
            best = by.unflatten(-1, (groups, -1)).sort(-1, descending=True).values[..., :group_best]
            first = best[..., 0]
            merit = first + torch.where(best == -math.inf, 0.0, best)[..., 1:].sum(-1)
            kept = torch.zeros_like(merit, dtype=torch.bool).scatter_(
                -1, torch.sort(-merit, dim=-1, stable=True).indices[..., :top_groups], True)
            kept = kept.repeat_interleave(rank.shape[-1] // groups, -1)
        else:
            kept = torch.ones_like(out)
        # Those out of reach last, before them NaN, before those -inf.
        tier = torch.where(kept, last.long(), 2)
        order = torch.sort(-rank, dim=-1, stable=True).indices
        order = order.gather(-1, torch.sort(tier.gather(-1, order), dim=-1, stable=True).indices)
        chosen = order[..., :k]
    z = logits.float()
    if renormalize:
        logs = z.gather(-1, chosen)
        logs = logs if score == 'softmax' else F.logsigmoid(logs)
        none = (logs == -math.inf).all(-1, keepdim=True)
        w = torch.softmax(logs.masked_fill(none, 0.0), -1).masked_fill(none, 0.0)
        if score == 'softmax':
            # (A factor, not a choice: the NaN goes into the gradients too.)
            w = w * torch.where((z.isnan() | (z == math.inf)).any(-1, keepdim=True), math.nan, 1.0)
    elif score == 'softmax':
        none = (z == -math.inf).all(-1, keepdim=True)
        w = torch.softmax(z.masked_fill(none, 0.0), -1).masked_fill(none, 0.0).gather(-1, chosen)
    else:
        w = torch.sigmoid(z.gather(-1, chosen))
    return w * scale, chosen.to(torch.int32)


# ------------------------------------------------------------------ rows to the experts and back

def arrange(chosen: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(slots, offsets)`` for ``chosen`` (int32 or int64 expert numbers of any shape,
    up to 1024 experts): ``slots`` (int32, chosen's shape) is each choice's place among
    all in the order of their experts, those of one expert in their given order, and
    ``offsets`` (int32, num_experts + 1) bounds each expert's places, as
    ``expert_linear`` takes them. Choices outside ``[0, num_experts)`` hold the places from
    ``offsets[-1]`` on, where ``expert_linear`` gives zeros: so choices are dropped (or by
    slots outside ``[0, tokens k)``; the rows of their places are zeros then)."""
    if chosen.is_cuda:
        return _binding.module().arrange(chosen, num_experts)
    if chosen.dtype not in (torch.int32, torch.int64):
        raise ValueError('chosen must be int32 or int64 expert numbers')
    if not 1 <= num_experts <= _native.MAX_EXPERTS:
        raise ValueError(f'num_experts must be 1 to {_native.MAX_EXPERTS}')
    flat = chosen.reshape(-1).long()
    flat = torch.where((flat < 0) | (flat >= num_experts), num_experts, flat)
    order = torch.argsort(flat, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel())
    ends = torch.bincount(flat, minlength=num_experts + 1)[:num_experts].cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    return slots.view(chosen.shape).to(torch.int32), offsets.to(torch.int32)


def _check_slots(slots, tokens=None):
    if slots.ndim != 2 or slots.dtype != torch.int32 or not 1 <= slots.shape[1] <= _native.MAX_CHOICES:
        raise ValueError(f'slots must be [tokens, k] in int32, with k from 1 to {_native.MAX_CHOICES}')
    if tokens is not None and slots.shape[0] != tokens:
        raise ValueError(f'slots must have {tokens} rows')


def dispatch(x: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """The tokens' rows in their experts' order: ``rows[slots[t, j]] = x[t]``, ``[tokens
    k, width]`` from x ``[tokens, width]`` (fp32, bf16 or f16, any row stride) and the
    slots of ``arrange`` (each place once; a slot outside ``[0, tokens k)`` stands for no
    place, and a place that no slot names gets zeros). CUDA tensors run natively, forward and
    backward (a token's gradient is the sum of its rows', in fp32); CPU tensors take plain
    PyTorch."""
    if x.is_cuda:
        return _binding.module().dispatch(x, slots)
    if x.ndim != 2 or x.shape[1] == 0 or x.dtype not in _FLOATS:
        raise ValueError('x must be [tokens, width] in float32, float16 or bfloat16')
    _check_slots(slots, x.shape[0])
    # The token of each place; places that no slot names stay zero.
    flat = slots.reshape(-1).long()
    named = (flat >= 0) & (flat < flat.numel())
    tokens = torch.arange(x.shape[0]).repeat_interleave(slots.shape[1])
    return x.new_zeros(flat.numel(), x.shape[1]).index_copy(
        0, flat[named], x.float()[tokens[named]].to(x.dtype))


def combine(rows: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, *,
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The experts' results back at their tokens: ``out[t] = residual[t] + sum_j
    weights[t, j] rows[slots[t, j]]``, ``[tokens, width]`` from rows ``[tokens k,
    width]`` (fp32, bf16 or f16, any row stride), the slots of ``arrange`` and fp32
    weights ``[tokens, k]``; sums in fp32, in the order of j, rounded once. A slot outside
    ``[0, tokens k)`` adds nothing, and rows that no slot names get zero gradients. CUDA tensors
    run natively, forward and backward (gradients of rows, weights and residual);
    forward-mode tangents, traces and second differentiation raise. CPU tensors take
    plain PyTorch."""
    if rows.is_cuda:
        return _binding.module().combine(rows, slots, weights, residual)
    _check_slots(slots)
    if rows.ndim != 2 or rows.shape[1] == 0 or rows.shape[0] != slots.numel() or rows.dtype not in _FLOATS:
        raise ValueError(f'rows must be [{slots.numel()}, width] in float32, float16 or bfloat16')
    if weights.shape != slots.shape or weights.dtype != torch.float32:
        raise ValueError(f'weights must be float32 of shape {list(slots.shape)}')
    if residual is not None and (residual.shape != (slots.shape[0], rows.shape[1]) or residual.dtype != rows.dtype):
        raise ValueError(f"residual must have the rows' type and shape {[slots.shape[0], rows.shape[1]]}")
    named = (slots >= 0) & (slots < slots.numel())
    # A choice without a row: zeros on both sides of the product, so that neither a weight that is infinite nor
    # the row in its stead reaches a result or a gradient.
    mine = rows.float()[torch.where(named, slots, 0).long()].masked_fill(~named.unsqueeze(-1), 0.0)
    out = (mine * weights.masked_fill(~named, 0.0).unsqueeze(-1)).sum(1)
    return (out if residual is None else out + residual.float()).to(rows.dtype)
