"""Cross entropy of a linear head's logits on the HIP kernels, without keeping the logits; differentiable to any order.

LinearCEOp          loss of z = x weight^T + bias from tiles of z that never leave the kernel; saves each row's largest logit
                    and sum of exponentials.
  .backward         -> LinearCEBackwardOp, itself an autograd.Function.
LinearCEBackwardOp  (dx, dweight, dbias), a piece of the vocabulary at a time.

Second and higher derivatives have no kernel: they differentiate a PyTorch restatement of the backward map on the device,
which materialises the logits (as hip_sdpa does from the third order on). The reference's models form logits and loss in
PyTorch.
"""

from __future__ import annotations

import torch

from .. import _ops

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _backward_map(x, weight, bias, target, dloss, ignore: int, reduction: int):
    """(dx, dweight, dbias) as differentiable PyTorch ops in float32 or wider."""
    ct = torch.promote_types(x.dtype, torch.float32)
    V, D = weight.shape
    t = target.reshape(-1).long()
    kept = (t != ignore) & (t >= 0) & (t < V)
    xf = torch.where(kept.unsqueeze(1), x.to(ct).reshape(-1, D), 0)
    wf = weight.to(ct)
    z = xf @ wf.t()
    if bias is not None:
        z = z + bias.to(ct)
    onehot = torch.where(kept, t, -1).unsqueeze(1) == torch.arange(V, device=t.device)
    up = torch.where(kept, dloss.to(ct).reshape(-1).expand(t.shape[0]), 0)
    if reduction == 1:
        up = up / kept.sum().clamp(min=1)
    dz = (torch.softmax(z, 1) - onehot.to(ct)) * up.unsqueeze(1)
    return (dz @ wf).reshape(x.shape).to(x.dtype), (dz.t() @ xf).to(weight.dtype), dz.sum(0)


class LinearCEBackwardOp(torch.autograd.Function):
    """(x, weight, bias, target, stats, dloss, ...) -> (dx, dweight, dbias)."""

    @staticmethod
    def forward(ctx, x, weight, bias, target, stats, dloss, ignore, reduction, need):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, target, dloss)
        ctx.args = (ignore, reduction)
        return _ops._host().linear_ce_bwd(x, weight, bias, target, stats, dloss, ignore, reduction, *need)

    @staticmethod
    def backward(ctx, u, a, c):
        x, weight, bias, target, dloss = ctx.saved_tensors
        needs = ctx.needs_input_grad
        prim = (x, weight, bias, dloss)
        want = (needs[0], needs[1], needs[2], needs[5])
        keep = torch.is_grad_enabled()
        with torch.enable_grad():
            # aliases, so that each result is a partial derivative; without a graph to keep, leaves of their own
            alias = [t if not w else t.view_as(t) if keep else t.detach().requires_grad_(True) for t, w in zip(prim, want)]
            wrt = [t for t, w in zip(alias, want) if w]
            outs = _backward_map(alias[0], alias[1], alias[2], target, alias[3], *ctx.args)
            pairs = [(o, g.to(o.dtype)) for o, g in zip(outs, (u, a, c)) if g is not None and o.requires_grad]
            if not pairs or not wrt:
                return (None,) * 9
            grads = iter(torch.autograd.grad([o for o, _ in pairs], wrt, [g for _, g in pairs], create_graph=keep, allow_unused=True))
        gx, gw, gb, gl = (next(grads) if w else None for w in want)
        return gx, gw, gb, None, None, gl, None, None, None


class LinearCEOp(torch.autograd.Function):
    """(x, weight, bias, target, ignore, reduction) -> loss."""

    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore, reduction):
        loss, stats = _ops._host().linear_ce_fwd(x, weight, bias, target, ignore, reduction)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, target, stats)
        ctx.args = (ignore, reduction)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        if dloss is None:
            return (None,) * 6
        x, weight, bias, target, stats = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():
            grads = LinearCEBackwardOp.apply(x, weight, bias, target, stats, dloss, *ctx.args, need)
        else:
            grads = _ops._host().linear_ce_bwd(x, weight, bias, target, stats, dloss, *ctx.args, *need)
        return (*grads, None, None, None)


def hip_linear_cross_entropy(x, weight, target, bias=None, *, ignore_index: int = -100, reduction: str = "mean"):
    """Cross entropy of the logits x weight^T + bias against target, without materialising the logits.

    x (..., D), weight (V, D) and bias (V,) in one of float32, float16, bfloat16; target (...) int32 or int64. Returns
    float32: the mean over the rows whose target is not ignore_index (NaN if there are none, with zero gradients), their
    sum, or with reduction "none" each row's loss (0 where ignored). What an ignored row of x holds is not read. A target
    outside [0, V) that is not ignore_index gives that row a loss and a gradient of NaN and adds nothing to the other gradients
    (checking it here would wait for the GPU). Gradients are those of torch.nn.functional.cross_entropy over the same
    logits. First derivatives are kernels; higher ones materialise the logits in PyTorch. torch.func transforms and
    forward-mode AD are not provided.
    """
    what = "hip_linear_cross_entropy"
    _ops.check_matrix(x, "x", what)
    _ops.check_matrix(weight, "weight", what)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise AssertionError(f"{what}: x must be (..., D) and weight (V, D), got {tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] < 1 or not 1 <= weight.shape[1] <= _ops.MAX_ROW_WIDTH:
        raise AssertionError(f"{what} supports V >= 1 and 1 <= D <= {_ops.MAX_ROW_WIDTH}, got weight {tuple(weight.shape)}")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise AssertionError(f"{what}: weight must match x in dtype and device")
    if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype != x.dtype or bias.device != x.device):
        raise AssertionError(f"{what}: bias must be ({weight.shape[0]},) and match x in dtype and device")
    _ops.check_indexes(target, "target", x, what)
    if tuple(target.shape) != tuple(x.shape[:-1]):
        raise AssertionError(f"{what}: target must have shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if reduction not in _REDUCTIONS:
        raise AssertionError(f"{what}: reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    return LinearCEOp.apply(x, weight, bias, target, int(ignore_index), _REDUCTIONS[reduction])


__all__ = ["LinearCEOp", "LinearCEBackwardOp", "hip_linear_cross_entropy"]
