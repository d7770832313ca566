"""Distillation loss from a teacher's top logits on the CUDA kernel, with its gradient.

The head of DeltaPhaseModel (delta_phase/model.py:60-66, 101) yields (B, L, vocab) logits; the
teacher gives K (index, logit) pairs per token.  :func:`distill_loss` is the differentiable
loss per token, :func:`distill_loss_and_grad` both in one pass over the logits
(``DeltaPhaseModel.distill_step`` calls it).
"""
from __future__ import annotations

import math

import torch

from .. import _capi


def _rows(t):
    """Logits (..., V) as the kernel reads them: (tensor, B, L, sb, st) with unit stride over V;
    in place wherever the leading dimensions are two or fewer, or can be viewed as two."""
    if t.dim() > 3:
        t = t.reshape(math.prod(t.shape[:-2]), t.shape[-2], t.shape[-1])
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    if t.dim() == 3:
        return t, t.shape[0], t.shape[1], t.stride(0), t.stride(1)
    if t.dim() == 2:
        return t, 1, t.shape[0], 0, t.stride(0)
    return t, 1, 1, 0, 0


def _like(t):
    """An empty contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _check(student_logits, teacher_index, teacher_logits, temperature, weight):
    """Refuses what the kernel does not take; returns tau and the constants as it takes them."""
    if student_logits.dim() < 1 or student_logits.shape[-1] < 1:
        raise ValueError("student_logits must be (..., V)")
    lead = student_logits.shape[:-1]
    if teacher_index.dim() < 1 or teacher_index.shape != teacher_logits.shape or \
            teacher_index.shape[:-1] != lead or teacher_index.shape[-1] < 1:
        raise ValueError(f"teacher_index and teacher_logits must both be {tuple(lead)} + (K,)")
    _capi.check_sizes(math.prod(lead), student_logits.shape[-1], teacher_index.shape[-1])
    if teacher_index.dtype not in (torch.int64, torch.int32):
        raise TypeError("teacher_index must be int64 or int32")
    _capi.dtype_code(student_logits)
    _capi.dtype_code(teacher_logits)
    if isinstance(temperature, torch.Tensor):
        raise TypeError("temperature must be a number")
    tau = float(temperature)
    if not 1e-30 < tau < 1e30:
        raise ValueError("temperature must be positive and finite")
    if weight is not None:
        if weight.shape != lead:
            raise ValueError(f"weight must be {tuple(lead)}, got {tuple(weight.shape)}")
        if weight.dtype != torch.float32 or not weight.is_contiguous():
            weight = weight.to(torch.float32).contiguous()
    return tau, teacher_index.contiguous(), teacher_logits.contiguous(), weight


class DistillCudaFunction(torch.autograd.Function):
    """Autograd wrapper on arguments that distill_loss has checked: forward on dp_distill, which
    also leaves the rows' maxima and sums; backward on dp_distill_bwd, which makes the gradient
    of them and the logits."""

    @staticmethod
    def forward(ctx, student_logits, index, teacher, tau, weight):
        loss = torch.empty(student_logits.shape[:-1], device=student_logits.device, dtype=torch.float32)
        stats = loss.new_empty((loss.numel(), 4))
        _capi.distill(*_rows(student_logits), index, teacher, weight, tau, loss, stats=stats)
        ctx.save_for_backward(student_logits, index, teacher, weight, stats)
        ctx.tau = tau
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        if torch.is_grad_enabled():  # create_graph: the gradient is not differentiable itself
            return _backward_once(ctx, grad_loss)
        return _backward(ctx, grad_loss)


def _backward(ctx, grad_loss):
    logits, index, teacher, weight, stats = ctx.saved_tensors
    dz = _like(logits)
    _capi.distill_bwd(*_rows(logits), index, teacher, weight, stats, grad_loss.contiguous(), ctx.tau, dz)
    return dz, None, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def distill_loss(student_logits, teacher_index, teacher_logits, temperature=1.0, weight=None):
    """Per-token distillation loss from a teacher's top logits, differentiable in the student's:

    ``weight * tau^2 * KL(p || q)`` with q = softmax(student_logits / tau) over the V logits and
    p = softmax(teacher_logits / tau) over the token's K entries.

    student_logits (..., V) float32 / bfloat16 / float16 (any strides; a slice such as
    ``logits[:, :-1]`` is read in place); teacher_index (..., K) int64 or int32, an index outside
    0 .. V - 1 marks a padding entry, one that occurs twice counts twice; teacher_logits (..., K),
    -inf leaves an entry out; weight (...) or None (1).  A token of weight 0 or without entries has
    loss and gradient 0, whatever its logits are.  Returns (...) float32.  Limits: K <= 1024,
    V times the element size below 1 MiB.
    """
    recording = torch.is_grad_enabled()
    if recording and (teacher_logits.requires_grad or (weight is not None and weight.requires_grad)):
        raise ValueError("teacher_logits and weight are constants of the loss: detach them")
    tau, index, teacher, w = _check(student_logits, teacher_index, teacher_logits, temperature, weight)
    if recording and student_logits.requires_grad:
        return DistillCudaFunction.apply(student_logits, index, teacher, tau, w)
    loss = torch.empty(student_logits.shape[:-1], device=student_logits.device, dtype=torch.float32)
    _capi.distill(*_rows(student_logits), index, teacher, w, tau, loss)
    return loss


def distill_loss_and_grad(student_logits, teacher_index, teacher_logits, temperature=1.0, weight=None):
    """:func:`distill_loss` and the gradient of its sum over all tokens with respect to the
    logits, in one pass over them: ``(loss (...) float32, grad (..., V) of the logits' dtype)``.
    Nothing is recorded for autograd; ``logits.backward(grad)`` carries the gradient on."""
    with torch.no_grad():
        tau, index, teacher, w = _check(student_logits, teacher_index, teacher_logits, temperature, weight)
        loss = torch.empty(student_logits.shape[:-1], device=student_logits.device, dtype=torch.float32)
        dz = _like(student_logits)
        _capi.distill(*_rows(student_logits), index, teacher, w, tau, loss, dz=dz)
    return loss, dz
