"""Layer norm for training on the CUDA kernels: forward, backward and the reduction of the
parameters' gradients, optionally with the residual add in front of it.

The blocks normalise three times (norm1, norm_retrieved, norm2; delta_phase/layers.py:177-244),
norm2 right after the residual add ``x + out_proj(...)``: :func:`layer_norm` with ``residual``
is that pair in one pass, on the float32 residual stream that the blocks keep
(``_capi.layernorm`` is its inference form).
"""
from __future__ import annotations

import torch

from .. import _capi


def _f32(t):
    """A parameter as the kernels take it (a copy only where it is not float32 already)."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.float().contiguous()


def _dense(t):
    return t if t.is_contiguous() else t.contiguous()


class LayerNormCudaFunction(torch.autograd.Function):
    """Autograd wrapper: forward on dp_layernorm_fwd, backward on dp_layernorm_bwd.  Saves s
    (x without a residual) and the rows' mean and 1 / sigma."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, out_dtype):
        xc = _dense(x)
        y = torch.empty_like(xc) if out_dtype == x.dtype else torch.empty_like(xc, dtype=out_dtype)
        stats = torch.empty((2, x.numel() // x.shape[-1]), device=x.device, dtype=torch.float32)
        res = s = None
        if residual is not None:
            res = _dense(residual)
            s = torch.empty_like(res)
        _capi.layernorm_fwd(xc, _f32(weight), _f32(bias), eps, y, stats, residual=res, sum_out=s)
        ctx.dtypes = x.dtype, None if bias is None else bias.dtype
        # x itself where it is contiguous, so that a change of x before the backward pass is noticed
        if s is None:
            ctx.save_for_backward(xc, weight, stats)
            return y
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(s, weight, stats)
        return y, s

    @staticmethod
    def backward(ctx, grad_y, grad_s=None):
        if torch.is_grad_enabled():  # create_graph: the gradients are not differentiable themselves
            return _backward_once(ctx, grad_y, grad_s)
        return _backward(ctx, grad_y, grad_s)


def _backward(ctx, grad_y, grad_s):
    if grad_y is None and grad_s is None:
        return None, None, None, None, None, None
    s, weight, stats = ctx.saved_tensors
    x_dtype, bias_dtype = ctx.dtypes
    need_x, need_w, need_b, _, need_res, _ = ctx.needs_input_grad
    gw = gb = dx = dres = None
    if need_w:
        gw = stats.new_empty(s.shape[-1])
    if need_b:
        gb = stats.new_empty(s.shape[-1])
    if grad_y is None:  # s alone was used
        if need_w:
            gw.zero_()
        if need_b:
            gb.zero_()
        dx = grad_s.to(x_dtype) if need_x else None
        dres = grad_s if need_res else None
    else:
        if need_res:
            dres = torch.empty_like(s)
        # a float32 x has the residual's gradient
        shared = need_x and need_res and x_dtype == torch.float32
        if need_x and not shared:
            dx = torch.empty_like(s) if s.dtype == x_dtype else torch.empty_like(s, dtype=x_dtype)
        if not grad_y.is_contiguous():
            grad_y = grad_y.contiguous()
        if grad_s is not None and not grad_s.is_contiguous():
            grad_s = grad_s.contiguous()
        _capi.layernorm_bwd(s, grad_y, _f32(weight), stats, grad_s, dx, dres, gw, gb)
        if shared:
            dx = dres
    if gw is not None and weight.dtype != torch.float32:
        gw = gw.to(weight.dtype)
    if gb is not None and bias_dtype != torch.float32:
        gb = gb.to(bias_dtype)
    return dx, gw, gb, None, dres, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None, out_dtype=None):
    """LayerNorm over the last dimension, differentiable: y = LayerNorm(x), or with
    ``residual`` s = x + residual and ``(LayerNorm(s), s)``.

    x (..., d) float32 / bfloat16 / float16; weight, bias (d,) of any of these types, or None
    (1 and 0); residual: float32, x's shape; s is float32.  y has ``out_dtype`` (default: x's
    dtype).  Statistics and sums are float32.  The gradients of weight and bias are summed over
    the rows in a fixed order.  Differentiable once.  A backward pass that is captured into a
    CUDA graph needs, as any in torch, leaves that no eager graph still refers to.
    """
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least 1")
    d = x.shape[-1]
    _capi.check_sizes(d)
    _capi.dtype_code(x)
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype not in _capi._DTYPE_CODES:
        raise TypeError(f"unsupported out_dtype {out_dtype}")
    for t in (weight, bias):
        if t is not None:
            _capi.dtype_code(t)
            if t.shape != (d,):
                raise ValueError(f"weight and bias must be ({d},), got {tuple(t.shape)}")
    if residual is not None:
        if residual.dtype != torch.float32:
            raise TypeError("the residual stream must be float32")
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    return LayerNormCudaFunction.apply(x, weight, bias, float(eps), residual, out_dtype)
