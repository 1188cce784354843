"""Layer norm on the HIP kernels, differentiable to any order.

LayerNormOp          y = (x - mean) rstd weight + bias; saves mean and rstd.
  .backward          -> LayerNormBackwardOp, itself an autograd.Function, so that gradients taken with create_graph=True
                     stay differentiable (full second-order MAML).
LayerNormBackwardOp  (dx, dweight, dbias); its backward is the explicit double-backward kernel.

As with hip_sdpa, derivatives of order three and higher have no kernel: they differentiate a PyTorch restatement of the
backward map on the device. The reference's models take their norms from PyTorch.
"""

from __future__ import annotations

import torch

from .. import _ops


def _backward_map(x, weight, dy, eps: float):
    """(dx, dweight, dbias) as differentiable PyTorch ops in float32 or wider (orders three and higher only)."""
    ct = torch.promote_types(x.dtype, torch.float32)
    D = x.shape[-1]
    xf, df = x.to(ct).reshape(-1, D), dy.to(ct).reshape(-1, D)
    xc = xf - xf.mean(1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + eps)
    xh = xc * rstd
    gw = df if weight is None else df * weight.to(ct)
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return dx.reshape(x.shape).to(x.dtype), (df * xh).sum(0), df.sum(0)


class LayerNormBackwardOp(torch.autograd.Function):
    """(x, weight, dy, mean, rstd, ...) -> (dx, dweight, dbias); mean and rstd are functions of x, whose part in the
    derivative the kernel includes."""

    @staticmethod
    def forward(ctx, x, weight, dy, mean, rstd, eps, need, param):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, dy, mean, rstd)
        ctx.eps, ctx.param = eps, param
        return _ops._host().layer_norm_bwd(x, weight, dy, mean, rstd, eps, *need, param)

    @staticmethod
    def backward(ctx, u, a, c):
        x, weight, dy, mean, rstd = ctx.saved_tensors
        if u is None and a is None and c is None:
            return (None,) * 8
        need = ctx.needs_input_grad
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, dy, u, a, c)):
            gx, gw, gy = _differentiable_double_backward(x, weight, dy, u, a, c, ctx.eps)
        else:
            gx, gw, gy = _ops._host().layer_norm_bwd_bwd(x, weight, dy, mean, rstd, ctx.eps, u, a, c, need[0], need[1], need[2],
                                                         ctx.param)
            if gy is not None and gy.dtype != dy.dtype:
                gy = gy.to(dy.dtype)
        return gx, gw, gy, None, None, None, None, None


def _differentiable_double_backward(x, weight, dy, u, a, c, eps):
    """The VJP of _backward_map with a graph. Its inputs are aliased, so that each result is a partial derivative."""
    prim = tuple(t.view_as(t) if t is not None and t.requires_grad else t for t in (x, weight, dy))
    wrt = [t for t in prim if t is not None and t.requires_grad]
    if not wrt:
        return None, None, None
    pairs = [(o, g.to(o.dtype)) for o, g in zip(_backward_map(*prim, eps), (u, a, c)) if g is not None]
    pairs = [(o, g) for o, g in pairs if o.requires_grad]
    if not pairs:
        return None, None, None
    grads = iter(torch.autograd.grad([o for o, _ in pairs], wrt, [g for _, g in pairs], create_graph=True, allow_unused=True))
    return tuple(next(grads) if t is not None and t.requires_grad else None for t in prim)


class LayerNormOp(torch.autograd.Function):
    """(x, weight, bias, eps) -> y."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _ops._host().layer_norm_fwd(x, weight, bias, eps)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.eps = eps
        ctx.param = weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():
            return (*LayerNormBackwardOp.apply(x, weight, dy, mean, rstd, ctx.eps, need, ctx.param), None)
        return (*_ops._host().layer_norm_bwd(x, weight, dy, mean, rstd, ctx.eps, *need, ctx.param), None)


def hip_layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5):
    """Layer norm of x (..., D) over its last dimension: (x - mean) / sqrt(var + eps) * weight + bias.

    x is float32, float16 or bfloat16, D at most 16384; weight and bias (D,) are optional, of x's dtype or both float32
    beside 16-bit x. Returns x's dtype; statistics and sums are float32. Reverse-mode derivatives of any order (the first
    two are kernels); torch.func transforms and forward-mode AD are not provided.
    """
    what = "hip_layer_norm"
    _ops.check_matrix(x, "x", what)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _ops.MAX_NORM_WIDTH:
        raise AssertionError(f"{what} supports rows of 1 to {_ops.MAX_NORM_WIDTH} elements, got shape {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (x.shape[-1],):
            raise AssertionError(f"{name} must have shape {(x.shape[-1],)}, got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32) or t.device != x.device:
            raise AssertionError(f"{what}: {name} must be on {x.device} in {x.dtype} or float32, got {t.dtype} on {t.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise AssertionError(f"{what}: weight and bias must have one dtype")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise AssertionError(f"{what}: eps must be finite and not negative, got {eps}")
    return LayerNormOp.apply(x, weight, bias, eps)


__all__ = ["LayerNormOp", "LayerNormBackwardOp", "hip_layer_norm"]
