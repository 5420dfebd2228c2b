"""``layernorm_rows``: layer norm of every row of token-major activations, with autograd.  cpm_kernels/torch/layernorm.py:8-66
normalises the middle axis of (batch, hidden, seq) and applies the affine step separately; this is the form in front of a linear whose
activations are (tokens, hidden), the layout ``bmm(x, False, w, True)`` takes."""
from typing import Optional

import torch

from ._ext import ext

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def layernorm_rows(x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, rd_mean: bool = True) -> torch.Tensor:
    """Layer norm of ``x`` (..., n) over its last axis, times ``weight`` (n), plus ``bias`` (n) if given; ``rd_mean`` False leaves the
    mean in (the RMS form).  fp16, bf16 or fp32, the same type for all three; statistics in fp32.  Differentiable in x, weight and bias
    (once).  Any n >= 1 and any number of rows, none included.

    Calls may be captured into a CUDA graph, the backward pass too.  As with PyTorch's own operators, a backward pass is captured only
    while no graph of an earlier, uncaptured call on the same leaves is alive: PyTorch ties a leaf's gradient to the stream of that call."""
    dtype, device = x.dtype, x.device
    assert x.is_cuda and x.is_contiguous() and x.ndim >= 1 and dtype in _DTYPES
    n = x.size(-1)
    assert 1 <= n <= 2 ** 30 and x.numel() // n < 2 ** 31
    assert eps >= 0
    assert weight.device == device and weight.dtype == dtype and weight.shape == (n,) and weight.is_contiguous()
    assert bias is None or (bias.device == device and bias.dtype == dtype and bias.shape == (n,) and bias.is_contiguous())
    return ext.layernorm_rows(x, eps, weight, bias, rd_mean)
