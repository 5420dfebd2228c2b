"""``layernorm_rows``: layer norm of every row of token-major activations, with autograd.  cpm_kernels/torch/layernorm.py:8-66
normalises the middle axis of (batch, hidden, seq) and applies the affine step separately; this is the form in front of a linear whose
activations are (tokens, hidden), the layout ``bmm(x, False, w, True)`` takes."""
from typing import Optional

import torch

from . import _ext


def layernorm_rows(x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, rd_mean: bool = True) -> torch.Tensor:
    """Layer norm of ``x`` (..., n) over its last axis, times ``weight`` (n), plus ``bias`` (n) if given; ``rd_mean`` False leaves the
    mean in (the RMS form).  fp16, bf16 or fp32, the same type for all three; statistics in fp32.  Differentiable in x, weight and bias
    (once; forward-mode differentiation raises a RuntimeError).  Any n >= 1 and any number of rows, none included.

    Calls may be captured into a CUDA graph, the backward pass too.  As with PyTorch's own operators, a backward pass is captured only
    while no graph of an earlier, uncaptured call on the same leaves is alive: PyTorch ties a leaf's gradient to the stream of that call."""
    return _ext.ext.layernorm_rows(x, eps, weight, bias, rd_mean)
