"""Embedding lookup with a scale on the HIP kernels, and its gradient by sorted tokens; differentiable to any order in
reverse mode.

The lookup is linear in the table: the gradient's own derivative is another lookup, so that no order needs a kernel of its
own. The autograd Functions are C++ (theria_amd/csrc/host/theria_host.cpp). The reference's models take their embeddings
from PyTorch.
"""

from __future__ import annotations

from .. import _ops


def hip_embedding(ids, weight, *, scale: float = 1.0, padding_idx: int | None = None):
    """Rows of weight (V, D) looked up by ids (int32 or int64, any shape), times scale: (*ids.shape, D) in weight's dtype.

    The gradient is a dense (V, D) table, summed in float32 in the tokens' order (the same bits on every run). The row of
    padding_idx is looked up like any other and gets no gradient. An id outside [0, V) gives a row of NaN and adds nothing to
    the gradient (checking it here would wait for the GPU). Reverse-mode derivatives of any order; torch.func transforms
    and forward-mode AD are not provided (they raise).
    """
    return _ops._host().embedding(ids, weight, scale, padding_idx)


__all__ = ["hip_embedding"]
