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
    """(..., n) as (B, L, n): a view wherever the leading dimensions allow it."""
    if t.dim() == 1:
        return t.view(1, 1, -1)
    return t.unsqueeze(0) if t.dim() == 2 else t.reshape(math.prod(t.shape[:-2]), t.shape[-2], t.shape[-1])


def _prepare(student_logits, teacher_index, teacher_logits, temperature, weight):
    if student_logits.dim() < 1 or student_logits.shape[-1] < 1:
        raise ValueError("student_logits must be (..., V)")
    lead = student_logits.shape[:-1]
    if teacher_index.dim() < 1 or teacher_index.shape != teacher_logits.shape or \
            teacher_index.shape[:-1] != lead or teacher_index.shape[-1] < 1:
        raise ValueError(f"teacher_index and teacher_logits must both be {tuple(lead)} + (K,)")
    if teacher_index.dtype not in (torch.int64, torch.int32):
        raise TypeError("teacher_index must be int64 or int32")
    _capi.dtype_code(student_logits)
    _capi.dtype_code(teacher_logits)
    if weight is not None and weight.shape != lead:
        raise ValueError(f"weight must be {tuple(lead)}, got {tuple(weight.shape)}")
    if isinstance(temperature, torch.Tensor):
        raise TypeError("temperature must be a number")
    tau = float(temperature)
    if not (tau > 0.0 and math.isfinite(tau)):
        raise ValueError("temperature must be positive and finite")
    _capi.require_cuda(student_logits, teacher_index, teacher_logits, weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (teacher_logits, weight)):
        raise ValueError("teacher_logits and weight are constants of the loss: detach them")
    z = _rows(student_logits.detach())
    if z.shape[-1] > 1 and z.stride(-1) != 1:
        z = z.contiguous()
    w = None if weight is None else weight.detach().to(torch.float32).contiguous()
    return z, _rows(teacher_index).contiguous(), _rows(teacher_logits.detach()).contiguous(), tau, w


class DistillCudaFunction(torch.autograd.Function):
    """Autograd wrapper of dp_distill: the loss in the forward pass; the backward pass reads the
    logits again and writes their gradient."""

    @staticmethod
    def forward(ctx, student_logits, teacher_index, teacher_logits, temperature, weight):
        z, idx, t, tau, w = _prepare(student_logits, teacher_index, teacher_logits, temperature, weight)
        loss = torch.empty(student_logits.shape[:-1], device=z.device, dtype=torch.float32)
        _capi.distill(z, idx, t, w, None, tau, loss=loss)
        ctx.save_for_backward(student_logits, teacher_index, teacher_logits, weight)
        ctx.tau = tau
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, index, teacher, weight = ctx.saved_tensors
        z, idx, t, tau, w = _prepare(logits, index, teacher, ctx.tau, weight)
        dz = torch.empty(logits.shape, device=z.device, dtype=z.dtype)
        _capi.distill(z, idx, t, w, grad_loss.to(torch.float32).contiguous(), tau, dz=dz)
        return dz, None, None, None, None


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
    if torch.is_grad_enabled() and student_logits.requires_grad:
        # the constants are looked at here: inside the function gradients are off
        _prepare(student_logits, teacher_index, teacher_logits, temperature, weight)
        return DistillCudaFunction.apply(student_logits, teacher_index, teacher_logits, temperature, weight)
    z, idx, t, tau, w = _prepare(student_logits, teacher_index, teacher_logits, temperature, weight)
    loss = torch.empty(student_logits.shape[:-1], device=z.device, dtype=torch.float32)
    _capi.distill(z, idx, t, w, None, tau, loss=loss)
    return loss


def distill_loss_and_grad(student_logits, teacher_index, teacher_logits, temperature=1.0, weight=None):
    """:func:`distill_loss` and the gradient of its sum over all tokens with respect to the
    logits, in one pass over them: ``(loss (...) float32, grad (..., V) of the logits' dtype)``.
    Nothing is recorded for autograd; ``logits.backward(grad)`` carries the gradient on."""
    with torch.no_grad():
        z, idx, t, tau, w = _prepare(student_logits, teacher_index, teacher_logits, temperature, weight)
        loss = torch.empty(student_logits.shape[:-1], device=z.device, dtype=torch.float32)
        dz = torch.empty(student_logits.shape, device=z.device, dtype=z.dtype)
        _capi.distill(z, idx, t, w, None, tau, loss=loss, dz=dz)
    return loss, dz
