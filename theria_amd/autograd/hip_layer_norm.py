"""Layer norm on the HIP kernels, differentiable to any order in reverse mode.

The autograd Functions are C++ (theria_amd/csrc/host/theria_host.cpp): the forward kernel, the backward kernel, whose
Function is itself differentiable so that gradients taken with create_graph=True stay in the graph (full second-order
MAML), and the explicit double-backward kernel. As with hip_sdpa, derivatives of order three and higher have no kernel: they
differentiate a restatement of the backward map in torch operations on the device. The reference's models take their norms
from PyTorch.
"""

from __future__ import annotations

from .. import _ops


def hip_layer_norm(x, weight=None, bias=None, *, eps: float = 1e-5):
    """Layer norm of x (..., D) over its last dimension: (x - mean) / sqrt(var + eps) * weight + bias.

    x is float32, float16 or bfloat16, D at most 16384; weight and bias (D,) are optional, of x's dtype or both float32
    beside 16-bit x. Returns x's dtype; statistics and sums are float32. Reverse-mode derivatives of any order (the first
    two are kernels); torch.func transforms and forward-mode AD are not provided (they raise).
    """
    return _ops._host().layer_norm(x, weight, bias, eps)


__all__ = ["hip_layer_norm"]
