"""Norm of each query and key head and rotation by position in one pass."""
from __future__ import annotations

import torch

from .. import ops

_OP = ops.head_norm_rotary.default


def rotary_table(positions, rotary_dim, base=10000.0, device="cuda"):
    """fp32 ``[positions, rotary_dim]``: row p holds cos(p w_i), then sin(p w_i),
    w_i = base^(-2 i / rotary_dim), computed in fp64 and rounded once."""
    if positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_table needs a position and an even rotary dimension")
    w = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * w
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def head_norm_rotary(q, k, table, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    """Norm of every head of ``q`` and ``k``, then the rotation by position.

    ``q`` ``[tokens, heads, dim]`` and ``k`` ``[tokens, kv_heads, dim]``, or
    both with a leading batch dimension (fp32, bf16 or fp16; any strides with
    contiguous heads, so views of a fused QKV projection and
    ``[batch, heads, sequence, dim]`` tensors transposed to this order need no
    copy; others are copied first); ``dim`` even and at most 512.
    ``positions`` int32 or int64
    ``[tokens]``, or ``[sequence]`` or ``[batch, sequence]``; ``table`` from
    ``rotary_table``, whose width is the rotated part of a head: pairs
    ``(i, i + rotary/2)``, or ``(2i, 2i + 1)`` when ``interleaved``. With
    weights ``[dim]`` (the heads' dtype or fp32) each head is first scaled by
    ``rsqrt(mean(x^2) + eps)`` and the weight; without, only turned. A position
    outside the table turns the rotated elements to NaN. Returns contiguous
    tensors of the shapes of ``q`` and ``k``; differentiable in ``q``, ``k``
    and the weights."""
    if not q.is_cuda:
        raise ValueError("head_norm_rotary requires CUDA tensors")
    return _OP(q, k, table, positions, q_weight, k_weight, eps, interleaved)
