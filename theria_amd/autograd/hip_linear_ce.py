"""Cross entropy of a linear head's logits on the HIP kernels, without keeping the logits; differentiable to any order in
reverse mode.

The forward forms tiles of the logits that never leave the kernel and keeps each row's largest logit and sum of
exponentials; the backward forms them again, a piece of the vocabulary at a time. The autograd Functions are C++
(theria_amd/csrc/host/theria_host.cpp). Second and higher derivatives have no kernel: they differentiate a restatement of the
backward map in torch operations on the device, which materialises the logits (as hip_sdpa does from the third order on).
The reference's models form logits and loss in PyTorch.
"""

from __future__ import annotations

from .. import _ops


def hip_linear_cross_entropy(x, weight, target, bias=None, *, ignore_index: int = -100, reduction: str = "mean"):
    """Cross entropy of the logits x weight^T + bias against target, without materialising the logits.

    x (..., D), weight (V, D) and bias (V,) in one of float32, float16, bfloat16; target (...) int32 or int64. Returns
    float32: the mean over the rows whose target is not ignore_index (NaN if there are none, with zero gradients), their
    sum, or with reduction "none" each row's loss (0 where ignored). What an ignored row of x holds is not read. A target
    outside [0, V) that is not ignore_index gives that row a loss and a gradient of NaN and adds nothing to the other gradients
    (checking it here would wait for the GPU). Gradients are those of torch.nn.functional.cross_entropy over the same
    logits. First derivatives are kernels; higher ones materialise the logits in PyTorch. torch.func transforms and
    forward-mode AD are not provided (they raise).
    """
    return _ops._host().linear_cross_entropy(x, weight, target, bias, ignore_index, reduction)


__all__ = ["hip_linear_cross_entropy"]
