"""Linear layers grouped by expert with ragged row counts.

``expert_linear(x, weight, offsets, bias)`` multiplies the rows
``[offsets[e], offsets[e + 1])`` of x by expert e's weights: the position-wise
layers of a mixture of experts (``layers.residual_linear`` is the dense form),
native in both directions (``avey_linear_fwd_v1``, ``avey_linear_bwd_v1``).
``group_by_expert`` sorts tokens for it. Row counts stay on the device:
neither call waits for the GPU, so both can be captured in a CUDA graph.

The reference has no counterpart ("Avey-B's static layers are ordinary matrix
multiplications and are outside this module", avey_kernels/ops.py:1-7).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from . import _binding, _native
from .layers import _ACT_IDS, _act_torch, _check_act


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
