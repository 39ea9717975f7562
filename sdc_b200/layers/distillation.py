"""Distillation loss against a teacher's top logits."""
from __future__ import annotations

import math

import torch

from .. import ops

_LOSS, _LOSS_AND_GRAD = ops.distillation_loss.default, ops.distill_loss_and_grad.default
_LOSS_AND_GRAD_IN_PLACE = ops.distill_loss_and_grad_.default
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _arguments(student_logits, teacher_indices, teacher_logits, temperature):
    if not student_logits.is_cuda:
        raise ValueError("distillation requires CUDA tensors")
    temperature = float(temperature)
    if not math.isfinite(temperature) or temperature <= 0:
        raise ValueError("distillation temperature must be positive and finite")
    if student_logits.dim() < 2 or teacher_indices.shape[:-1] != student_logits.shape[:-1] or \
            teacher_logits.shape != teacher_indices.shape:
        raise ValueError("distillation needs logits [..., vocabulary] and teacher indices and logits [..., top]")
    if student_logits.dim() > 2:
        teacher_indices = teacher_indices.flatten(0, -2)
        teacher_logits = teacher_logits.flatten(0, -2)
        student_logits = student_logits.flatten(0, -2)
    return student_logits, teacher_indices, teacher_logits, temperature


def distillation_loss(student_logits, teacher_indices, teacher_logits, temperature=1.0, reduction="mean"):
    """KL divergence of the teacher's distribution over its top tokens from the
    student's over the whole vocabulary, times ``temperature^2``.

    ``student_logits`` ``[..., vocabulary]`` (fp32, bf16 or fp16, any row
    stride; column-major ones are copied to rows first); ``teacher_indices``
    (int32 or int64) and ``teacher_logits`` ``[..., top]`` with ``top`` up to
    1024. Both distributions are softmaxes at the temperature, the teacher's
    over its list alone. Negative indices are no
    entries; entries that name a token twice add up; a row without entries (or
    with teacher logits of -inf alone) has loss 0 and gradient 0 whatever its
    student logits; an index beyond the vocabulary makes the row NaN.

    ``reduction``: "none" (fp32, one loss a row), "sum", or "mean" over the
    rows that have entries. Differentiable in the student's logits (a teacher's
    that require a gradient are refused: ``detach()`` them); the backward pass
    reads them again. Where the upstream gradient is known
    beforehand, ``distillation_loss_and_grad`` reads them once."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}")
    shape = student_logits.shape[:-1]
    student, indices, teacher, temperature = _arguments(student_logits, teacher_indices, teacher_logits, temperature)
    loss = _LOSS(student, indices, teacher, temperature, _REDUCTIONS[reduction])
    return loss.view(shape) if reduction == "none" and len(shape) != 1 else loss


@torch.no_grad()
def distillation_loss_and_grad(student_logits, teacher_indices, teacher_logits, temperature=1.0, grad_loss=None,
                               in_place=False):
    """The losses of every row (as ``reduction="none"``) and the gradient of
    ``sum(grad_loss * losses)`` with respect to the logits, in one pass over
    them. ``grad_loss``: fp32 scalar tensor or one value a row; None: 1. With
    ``in_place`` the gradient replaces the logits (contiguous rows). Not
    recorded by autograd: hand the gradient to
    ``torch.autograd.backward(logits, grad)``."""
    shape = student_logits.shape
    student, indices, teacher, temperature = _arguments(student_logits, teacher_indices, teacher_logits, temperature)
    if grad_loss is not None and grad_loss.dim() > 1:
        if grad_loss.shape != shape[:-1]:
            raise ValueError("grad_loss must be a scalar or have one value a row")
        grad_loss = grad_loss.reshape(-1)
    if in_place:
        if student.data_ptr() != student_logits.data_ptr():
            raise ValueError("in-place distillation needs logits whose rows flatten without a copy")
        loss, grad = _LOSS_AND_GRAD_IN_PLACE(student, indices, teacher, temperature, grad_loss), student
    else:
        loss, grad = _LOSS_AND_GRAD(student, indices, teacher, temperature, grad_loss)
    return loss.view(shape[:-1]), grad.view(shape)
