"""Gated linear recurrence on the CUDA kernels: h_t = a_t h_{t-1} + u_t per channel.

The vector-state counterpart of LaplacePhaseCore's per-row decay (delta_phase/layers.py:481-561):
:func:`gated_scan` runs a whole sequence (differentiable), :func:`gated_scan_step` one decode
token, like ``laplace_chunkwise`` and ``decode_step`` do for the matrix states.
"""
from __future__ import annotations

import torch

from .. import _capi

_MODES = {"decay": _capi.DP_SCAN_DECAY, "sigmoid": _capi.DP_SCAN_SIGMOID}


def _mode(gate_mode):
    try:
        return _MODES[gate_mode]
    except (KeyError, TypeError):
        raise ValueError(f"gate_mode must be one of {sorted(_MODES)}, got {gate_mode!r}") from None


def _like(t):
    """An empty contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, device=t.device, dtype=t.dtype)


def _unit(t):
    """t with unit channel stride (a copy only where it has none)."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _seq(t):
    """A (B, L, D) tensor as the kernels read it: unit channel stride, token strides within their
    32 bits (a copy where it has neither)."""
    t = _unit(t)
    if t.stride(1) > _capi.SCAN_MAX_TOKEN_STRIDE:
        t = t.contiguous()
        if t.stride(1) > _capi.SCAN_MAX_TOKEN_STRIDE:  # one token: its stride moves nothing
            t = t.as_strided(t.shape, (t.stride(0), t.shape[2], 1))
    return t


def _check_inputs(x, gate, dims, what):
    if x.dim() != dims or gate.shape != x.shape or x.shape[-1] < 1:
        raise ValueError(f"x and gate must both be {what}")
    _capi.check_sizes(*x.shape)
    _capi.dtype_code(x)
    if gate.dtype != x.dtype:
        raise TypeError("x and gate must share one dtype")


def _check_state(state, B, D, name):
    if state.dtype != torch.float32:
        raise TypeError(f"{name} must be float32")
    if tuple(state.shape) != (B, D):
        raise ValueError(f"{name} must be (B, D) = {(B, D)}, got {tuple(state.shape)}")


def _forward(x, gate, initial_state, mode, keep):
    B, L, D = x.shape
    h0 = None if initial_state is None else initial_state.contiguous()
    out = _like(x)
    final = torch.empty((B, D), device=x.device, dtype=torch.float32)
    saved = None
    if keep:
        tile = _capi.scan_tile()
        saved = final.new_empty((B, (L + tile - 1) // tile, D))
    _capi.scan_fwd(_seq(x), _seq(gate), mode, h0, _seq(out), final, saved)
    return out, final, saved


class GatedScanCudaFunction(torch.autograd.Function):
    """Autograd wrapper: forward on dp_scan_fwd, backward on dp_scan_bwd.  Saves the inputs and
    the float32 state before every tile of tokens; the backward recomputes the states between."""

    @staticmethod
    def forward(ctx, x, gate, initial_state, mode):
        out, final, saved = _forward(x, gate, initial_state, mode, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, gate, saved)
        ctx.mode = mode
        return out, final

    @staticmethod
    def backward(ctx, grad_out, grad_final):
        if torch.is_grad_enabled():  # create_graph: the gradients are not differentiable themselves
            return _backward_once(ctx, grad_out, grad_final)
        return _backward(ctx, grad_out, grad_final)


def _backward(ctx, grad_out, grad_final):
    x, gate, saved = ctx.saved_tensors
    if grad_out is None and grad_final is None:
        return None, None, None, None
    need_x, need_gate, need_state, _ = ctx.needs_input_grad
    dx, dg = _like(x), _like(x)
    go = torch.zeros_like(dx) if grad_out is None else _seq(grad_out)
    gf = None if grad_final is None else grad_final.contiguous()
    dh = saved.new_empty((x.shape[0], x.shape[2])) if need_state else None
    _capi.scan_bwd(_seq(x), _seq(gate), go, ctx.mode, saved, gf, dx, dg, dh)
    return dx if need_x else None, dg if need_gate else None, dh, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def gated_scan(x, gate, initial_state=None, gate_mode="decay"):
    """Gated linear recurrence over a sequence, per channel, from ``initial_state`` (zero):

    * ``gate_mode="decay"``:   h_t = exp(gate_t) h_{t-1} + x_t  (gate = log a; -inf drops the
      state, e.g. at the first token of a packed document)
    * ``gate_mode="sigmoid"``: h_t = sigmoid(gate_t) h_{t-1} + (1 - sigmoid(gate_t)) x_t

    x, gate (B, L, D) of one dtype (float32 / bfloat16 / float16; any strides, without a copy
    where the channel stride is 1 and tokens are at most 2^28 elements apart); initial_state (B, D) float32 or None, never modified.  Any L up to 2^30.
    Returns ``(out (B, L, D) of x's dtype, h_L (B, D) float32)``; the state is float32
    throughout and the order of all sums depends on L alone.  A value that is not finite stays in
    its channel, from its token on (an infinite state may continue as NaN).  Differentiable once when autograd
    records and an input requires grad.  A backward pass that is captured into a CUDA graph
    needs, as any in torch, leaves that no eager graph still refers to.  Like the other kernels whose
    blocks wait for one another, these give a wait up after 2 s and report it through
    ``_capi.device_error()``, not through this call; the results are not to be used then.
    """
    mode = _mode(gate_mode)
    _check_inputs(x, gate, 3, "(B, L, D)")
    if initial_state is not None:
        _check_state(initial_state, x.shape[0], x.shape[2], "initial_state")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, initial_state)):
        return GatedScanCudaFunction.apply(x, gate, initial_state, mode)
    return _forward(x, gate, initial_state, mode, False)[:2]


def gated_scan_step(state, x, gate, gate_mode="decay", state_out=None, out=None):
    """One token of :func:`gated_scan`: state (B, D) float32, x and gate (B, D).  Returns
    ``(out (B, D) of x's dtype, new_state)``; ``state_out=state`` updates the state in place.  An
    output may lie on another tensor of its type element for element, but not overlap it otherwise.
    Not differentiable (like ``decode_step``)."""
    mode = _mode(gate_mode)
    _check_inputs(x, gate, 2, "(B, D)")
    B, D = x.shape
    _check_state(state, B, D, "state")
    given = [t for t in (state_out, out) if t is not None]
    if state_out is None:
        state_out = _like(state)
    else:
        _check_state(state_out, B, D, "state_out")
        if not state_out.is_contiguous():
            raise ValueError("state_out must be contiguous")
    if out is None:
        out = _like(x)
    elif out.dtype != x.dtype or out.shape != x.shape or (D > 1 and out.stride(1) != 1) or \
            (B > 1 and out.stride(0) < D):
        raise ValueError("out must be a (B, D) tensor of x's dtype with unit channel stride and rows apart")
    _capi.scan_step(state.contiguous(), state_out, _unit(x), _unit(gate), mode, out)
    if given:  # autograd notices a change of what it has saved
        torch.autograd.graph.increment_version(given)
    return out, state_out
