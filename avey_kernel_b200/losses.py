"""Losses over a vocabulary that never hold its logits.

``linear_cross_entropy(x, weight, targets)`` is the end of a language model: the
head's product ``z = x W^T`` and the softmax cross entropy of it in one operator
(``avey_loss_fwd_v1``, ``avey_loss_bwd_v1``). ``z`` exists only tile by tile in
the tensor cores' memory: the forward pass keeps one number a row, the backward
pass computes z again in pieces of the vocabulary.

The reference has no counterpart: it leaves the head and the loss to torch.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import _binding, _native


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = 'mean', z_loss: float = 0.0
                         ) -> torch.Tensor:
    """Softmax cross entropy of ``x W^T`` against ``targets``, in fp32.

    x ``[..., width]``, weight ``[vocab, width]`` (``nn.Linear`` layout), targets
    ``[...]`` (int64 or int32). For a row with log sum ``lse = log sum_j exp z_j``::

        loss = lse - z_target + z_loss lse^2

    and 0 where the target is ``ignore_index``: such rows have no part in the loss
    or the gradients, whatever x holds there, and ``z_loss`` (usually about 1e-4)
    keeps the log sums near zero. ``reduction`` is 'none' (losses of targets'
    shape), 'sum' or 'mean' (over the rows that are not ignored; NaN when all are).
    A target outside the vocabulary makes its row's loss NaN, and with it the row's gradient and
    the weight's.

    Memory beside the tensors and their gradients: the backward pass takes up to 512 MB
    for pieces of the logits' gradient (16 KB a row above 32768 rows) and 6 bytes for
    every element of x; rows that are not whole 16-byte units (of widths that 8 does not
    divide, or views off 16 bytes) are copied in either pass, x's and the weight's.

    bf16 / f16 CUDA tensors of one dtype run natively, forward and backward, with
    any row strides: fp32 sums, the gradient at the logits rounded to the operand
    type before its two products (relative to the largest gradient that comes in, so
    that f16 keeps small probabilities), and each result rounded once. Tensors with
    forward-mode tangents, calls under a trace (``torch.jit.trace``, ``make_fx``) and
    second differentiation raise. CPU tensors take plain PyTorch."""
    if reduction not in _native.REDUCTION_IDS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    if x.is_cuda:
        return _binding.module().cross_entropy(x, weight, targets, ignore_index,
                                               _native.REDUCTION_IDS[reduction], z_loss)
    if weight.dtype != x.dtype or x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError('x and weight must be float32, float16 or bfloat16 of one dtype')
    if x.ndim < 1 or weight.ndim != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError('x must be [..., width] and weight [vocab, width]')
    if targets.shape != x.shape[:-1]:
        raise ValueError(f'targets must have shape {list(x.shape[:-1])}')
    if targets.dtype not in (torch.int32, torch.int64):
        raise ValueError('targets must be int32 or int64')
    if not math.isfinite(z_loss):
        raise ValueError('z_loss must be finite')
    return _cross_entropy_torch(x, weight, targets, ignore_index, reduction, z_loss)


def _cross_entropy_torch(x, weight, targets, ignore_index, reduction, z_loss):
    """The plain PyTorch form (CPU tensors)."""
    used = targets != ignore_index
    inside = (targets >= 0) & (targets < weight.shape[0])
    z = F.linear(x.masked_fill(~used.unsqueeze(-1), 0).float(), weight.float())
    # (log_softmax subtracts the largest logit first: the log sum would be rounded at its size.)
    each = -F.log_softmax(z, dim=-1).gather(-1, torch.where(inside, targets, 0).long().unsqueeze(-1)).squeeze(-1)
    if z_loss != 0.0:
        each = each + z_loss * torch.logsumexp(z, dim=-1).square()
    # (A factor, not a choice: the NaN of a bad target goes into the gradients too.)
    each = torch.where(used, each * torch.where(used & ~inside, math.nan, 1.0), 0.0)
    if reduction == 'none':
        return each
    return each.sum() if reduction == 'sum' else each.sum() / used.sum()
