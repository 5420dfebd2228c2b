"""``layernorm_rows``: layer norm of every row of token-major activations, with autograd.  cpm_kernels/torch/layernorm.py:8-66
normalises the middle axis of (batch, hidden, seq) and applies the affine step separately; this is the form in front of a linear whose
activations are (tokens, hidden), the layout ``bmm(x, False, w, True)`` takes."""
from typing import Optional

import torch

from ..kernels import layernorm_rows_forward, layernorm_rows_backward, layernorm_rows_backward_scratch
from ..library import cpmk

_DTYPES = {torch.float16: cpmk.F16, torch.bfloat16: cpmk.BF16, torch.float32: cpmk.F32}


def _forward(x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor], rd_mean: bool, statistics: bool):
    n = x.size(-1)
    rows = x.numel() // n
    y = torch.empty_like(x)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if statistics else None
    with torch.cuda.device(x.device):
        layernorm_rows_forward(rows, n, _DTYPES[x.dtype], x.data_ptr(), eps, rd_mean, weight.data_ptr(), bias.data_ptr() if bias is not None else 0,
                               y.data_ptr(), stats[0].data_ptr() if statistics else 0, stats[1].data_ptr() if statistics else 0,
                               torch.cuda.current_stream().cuda_stream)
    return y, stats


class OpLayerNormRows(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor], rd_mean: bool):
        y, stats = _forward(x, eps, weight, bias, rd_mean, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.rd_mean = rd_mean
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output: torch.Tensor):
        x, weight, stats = ctx.saved_tensors
        dy = grad_output.contiguous()
        n = x.size(-1)
        rows = x.numel() // n
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        dweight = torch.empty_like(weight) if ctx.needs_input_grad[2] else None
        dbias = torch.empty_like(weight) if ctx.needs_input_grad[3] else None
        with torch.cuda.device(x.device):
            scratch = torch.empty((layernorm_rows_backward_scratch(rows, n),), dtype=torch.uint8, device=x.device)
            layernorm_rows_backward(rows, n, _DTYPES[x.dtype], dy.data_ptr(), x.data_ptr(), ctx.rd_mean, weight.data_ptr(), stats[0].data_ptr(),
                                    stats[1].data_ptr(), dx.data_ptr() if dx is not None else 0, dweight.data_ptr() if dweight is not None else 0,
                                    dbias.data_ptr() if dbias is not None else 0, scratch.data_ptr(), torch.cuda.current_stream().cuda_stream)
        return dx, None, dweight, dbias, None


def layernorm_rows(x: torch.Tensor, eps: float, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, rd_mean: bool = True) -> torch.Tensor:
    """Layer norm of ``x`` (..., n) over its last axis, times ``weight`` (n), plus ``bias`` (n) if given; ``rd_mean`` False leaves the
    mean in (the RMS form).  fp16, bf16 or fp32, the same type for all three; statistics in fp32.  Differentiable in x, weight and bias
    (once).  Any n >= 1 and any number of rows, none included."""
    assert x.is_cuda and x.is_contiguous() and x.ndim >= 1 and x.dtype in _DTYPES
    assert x.size(-1) >= 1 and x.numel() // x.size(-1) < 2 ** 31
    assert eps >= 0
    for v in (weight, bias):
        if v is not None:
            assert v.is_cuda and v.device == x.device and v.is_contiguous() and v.ndim == 1 and v.dtype == x.dtype and v.numel() == x.size(-1)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return OpLayerNormRows.apply(x, eps, weight, bias, rd_mean)
    return _forward(x, eps, weight, bias, rd_mean, False)[0]
