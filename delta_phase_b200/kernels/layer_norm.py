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
    return None if t is None else t.detach().float().contiguous()


class LayerNormCudaFunction(torch.autograd.Function):
    """Autograd wrapper: forward on dp_layernorm_fwd, backward on dp_layernorm_bwd.  Saves s
    (x without a residual) and the rows' mean and 1 / sigma."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual, out_dtype):
        d = x.shape[-1]
        x2 = x.detach().reshape(-1, d).contiguous()
        rows = x2.shape[0]
        dev = x.device
        y = torch.empty(rows, d, device=dev, dtype=out_dtype)
        stats = torch.empty(2, rows, device=dev, dtype=torch.float32)
        res = s = None
        if residual is not None:
            res = residual.detach().reshape(-1, d).contiguous()
            s = torch.empty(rows, d, device=dev, dtype=torch.float32)
        _capi.layernorm_fwd(x2, _f32(weight), _f32(bias), eps, y, stats[0], stats[1], residual=res, sum_out=s)
        ctx.set_materialize_grads(False)
        ctx.shape, ctx.x_dtype = x.shape, x.dtype
        ctx.has_residual = residual is not None
        ctx.bias_dtype = None if bias is None else bias.dtype
        y = y.view(x.shape)
        if residual is None:
            # x itself where it is contiguous, so that a change of x before the backward pass is noticed
            ctx.save_for_backward(x if x.is_contiguous() else x2, weight, stats)
            return y
        s = s.view(x.shape)
        ctx.save_for_backward(s, weight, stats)
        return y, s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_s=None):
        s, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _, need_res, _ = ctx.needs_input_grad
        shape, d = ctx.shape, ctx.shape[-1]
        if grad_y is None and grad_s is None:
            return None, None, None, None, None, None
        f32 = dict(device=s.device, dtype=torch.float32)
        s2 = s.reshape(-1, d)
        gs = None if grad_s is None else grad_s.reshape(-1, d).contiguous()
        if grad_y is None:
            gw = torch.zeros(d, **f32) if need_w else None
            gb = torch.zeros(d, **f32) if need_b else None
            dx = gs.to(ctx.x_dtype) if need_x else None
            dres = gs if need_res else None
        else:
            gw = torch.empty(d, **f32) if need_w else None
            gb = torch.empty(d, **f32) if need_b else None
            dres = torch.empty(s2.shape, **f32) if need_res else None
            # a float32 x has the residual's gradient
            shared = need_x and need_res and ctx.x_dtype == torch.float32
            dx = torch.empty(s2.shape, device=s.device, dtype=ctx.x_dtype) if need_x and not shared else None
            _capi.layernorm_bwd(s2, grad_y.reshape(-1, d).contiguous(), _f32(weight), stats[0], stats[1],
                                grad_sum=gs, dx=dx, grad_residual=dres, grad_w=gw, grad_b=gb)
            if shared:
                dx = dres
        return (None if dx is None else dx.view(shape),
                None if gw is None else gw.to(weight.dtype),
                None if gb is None else gb.to(ctx.bias_dtype), None,
                None if dres is None else dres.view(shape), None)


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
    out_dtype = x.dtype if out_dtype is None else out_dtype
    for t in (x, weight, bias):
        if t is not None:
            _capi.dtype_code(t)
    if out_dtype not in _capi._DTYPE_CODES:
        raise TypeError(f"unsupported out_dtype {out_dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (d,):
            raise ValueError(f"{name} must be ({d},), got {tuple(t.shape)}")
    if residual is not None:
        if residual.dtype != torch.float32:
            raise TypeError("the residual stream must be float32")
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    _capi.require_cuda(x, weight, bias, residual)
    return LayerNormCudaFunction.apply(x, weight, bias, float(eps), residual, out_dtype)
