"""Embedding lookup with a scale on the HIP kernels, and its gradient by sorted tokens; differentiable to any order.

The lookup is linear in the table: the gradient's own derivative is another lookup, so that no order needs a kernel of its
own. The reference's models take their embeddings from PyTorch.
"""

from __future__ import annotations

import math

import torch

from .. import _ops


class EmbeddingBackwardOp(torch.autograd.Function):
    """(dout, ids, ...) -> the table's gradient."""

    @staticmethod
    def forward(ctx, dout, ids, classes, scale, padding):
        ctx.save_for_backward(ids)
        ctx.args = (scale, padding)
        return _ops._host().embedding_bwd(ids, dout, classes, scale, padding)

    @staticmethod
    def backward(ctx, gtable):
        (ids,) = ctx.saved_tensors
        return EmbeddingOp.apply(gtable, ids, *ctx.args, True), None, None, None, None


class EmbeddingOp(torch.autograd.Function):
    """(table, ids, scale, padding, zero_padding) -> rows of the table times scale."""

    @staticmethod
    def forward(ctx, table, ids, scale, padding, zero_padding):
        ctx.save_for_backward(ids)
        ctx.args = (table.shape[0], scale, padding)
        return _ops._host().embedding_fwd(ids, table, scale, padding, zero_padding)

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        if torch.is_grad_enabled():
            return EmbeddingBackwardOp.apply(dout, ids, *ctx.args), None, None, None, None
        return _ops._host().embedding_bwd(ids, dout, *ctx.args), None, None, None, None


def hip_embedding(ids, weight, *, scale: float = 1.0, padding_idx: int | None = None):
    """Rows of weight (V, D) looked up by ids (int32 or int64, any shape), times scale: (*ids.shape, D) in weight's dtype.

    The gradient is a dense (V, D) table, summed in float32 in the tokens' order (the same bits on every run). The row of
    padding_idx is looked up like any other and gets no gradient. An id outside [0, V) gives a row of NaN and adds nothing to
    the gradient (checking it here would wait for the GPU). Reverse-mode derivatives of any order; torch.func transforms
    and forward-mode AD are not provided.
    """
    what = "hip_embedding"
    _ops.check_matrix(weight, "weight", what)
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= _ops.MAX_ROW_WIDTH:
        raise AssertionError(f"{what}: weight must be (V, D) with 1 <= D <= {_ops.MAX_ROW_WIDTH}, got shape {tuple(weight.shape)}")
    _ops.check_indexes(ids, "ids", weight, what)
    V = weight.shape[0]
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx)
        padding = padding + V if padding < 0 else padding
        if not 0 <= padding < V:
            raise AssertionError(f"{what}: padding_idx {padding_idx} is outside the table of {V} rows")
    scale = float(scale)
    if not math.isfinite(scale):
        raise AssertionError(f"{what}: scale must be finite, got {scale}")
    return EmbeddingOp.apply(weight, ids, scale, padding, False)


__all__ = ["EmbeddingOp", "EmbeddingBackwardOp", "hip_embedding"]
